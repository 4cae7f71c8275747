"""Operators of a model whose projections run in 8 bits (e4m3), as a serving program calls them, as cases to measure.

norm    the pending adds into the residual, then the root-mean-square norm of it, leaving codes of 8 bits and a scale for each row
rows    rows of activations (attention's output, the hidden units) to codes and a scale for each row
linear  a projection: codes of activations times codes of weights, the two scales, bias, activation and addend applied to the sum in 32 bits
gateup  the gate and up projections of a feed-forward block and the gated unit of their sums

A row x of codes c and scale s stands for c * s, s = (largest magnitude) / 448; weights have a scale for each output.  The norm's row is
(largest magnitude of x * weight) * rms factor / 448, so that its codes do not depend on the rms factor.
"""
import math
import os
import sys

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_E4M3 = torch.float8_e4m3fn
_LARGEST = 448.0         # of e4m3
_SMALLEST = 2.0 ** -100  # a row of smaller values than this is stored against it
_EPS = 1e-5


# ---- cases --------------------------------------------------------------------------------------------------------------------
def _norm(name, dtype, rows, dim, adds, factor=1.0):
    """`adds` pending addends of a residual that is scaled by `factor` first."""
    return {"name": name, "op": "norm", "dtype": dtype, "rows": rows, "dim": dim, "adds": adds, "factor": factor}


def _rows(name, dtype, rows, cols, apart=0):
    """Rows of `cols` elements, `apart` more elements between them (a part of a wider projection's output)."""
    return {"name": name, "op": "rows", "dtype": dtype, "rows": rows, "cols": cols, "apart": apart}


def _linear(name, dtype, rows, n, k, bias=False, act="none", addend=False):
    return {"name": name, "op": "linear", "dtype": dtype, "rows": rows, "n": n, "k": k, "bias": bias, "act": act, "addend": addend}


def _gateup(name, dtype, rows, inter, k, alpha=1.0, limit=math.inf, offset=0.0):
    return {"name": name, "op": "gateup", "dtype": dtype, "rows": rows, "inter": inter, "k": k, "alpha": alpha, "limit": str(limit), "offset": offset}


def listed():
    return [
        # one new token of the 8B shape: nothing but latency
        _norm("norm-1", "bf16", 1, 4096, 1),
        # a served batch in the type of the reference's driver, both partial sums pending, the residual divided among ranks
        _norm("norm-40-fp16", "fp16", 40, 2560, 2, 0.5),
        # a long prompt of the 8B shape
        _norm("norm-prompt-8k", "bf16", 8192, 4096, 1),
        # attention's output of a batch of 16, a part of a wider buffer
        _rows("rows-16", "bf16", 16, 4096, 2048),
        # the hidden units of a prompt, of a width that is no multiple of 16
        _rows("rows-prompt-odd", "fp16", 2047, 11000),
        # one new token through the query, key and value projection of the 8B shape
        _linear("linear-1-qkv", "bf16", 1, 6144, 4096),
        # a batch of 24 through the down projection of the 8B shape, added to what attention has left
        _linear("linear-24-down", "bf16", 24, 4096, 14336, addend=True),
        # a ragged batch through a projection with bias and activation, of sizes that are no multiples of a tile
        _linear("linear-333-bias-gelu", "fp16", 333, 2001, 2568, bias=True, act="gelu"),
        # a prompt through the output projection of the 70B shape, added to the residual
        _linear("linear-prompt-4k", "bf16", 4096, 8192, 8192, addend=True),
        # four users of the 8B shape
        _gateup("gateup-4", "bf16", 4, 14336, 4096),
        # a batch of 64 of the 1B shape, the clamped unit of the layer-list designs
        _gateup("gateup-64-clamped", "fp16", 64, 8192, 2048, 1.702, 7.0, 1.0),
        # a prompt of the 8B shape
        _gateup("gateup-prompt-4k", "bf16", 4096, 14336, 4096),
    ]


def draw(rng):
    def spread(lo, hi):
        return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))

    op, dtype = rng.choice(("norm", "rows", "linear", "linear", "gateup", "gateup")), rng.choice(("bf16", "fp16"))
    rows = spread(1, 4096)
    if op == "norm":
        c = _norm("", dtype, rows, 8 * spread(36, 1024), rng.choice((0, 1, 1, 2)), rng.choice((1.0, 1.0, 0.25)))
    elif op == "rows":
        c = _rows("", dtype, rows, 8 * spread(8, 2048), 8 * rng.choice((0, 0, spread(1, 512))))
    else:
        k = 8 * spread(36, 1792)
        n = spread(64, min(28672, 100_000_000 // k))
        if rng.random() < 0.6:
            n = -(-n // 64) * 64
        if op == "linear":
            c = _linear("", dtype, rows, n, k, rng.random() < 0.4, rng.choice(("none", "none", "silu", "gelu", "gelu_tanh")), rng.random() < 0.5)
        else:
            c = _gateup("", dtype, rows, (n + 1) // 2, k, *rng.choice(((), (), (1.702, 7.0, 1.0), (1.0, 4.0, 0.0))))
    del c["name"]
    return c


def work(case):
    m = case["rows"]
    if case["op"] == "norm":
        d = case["dim"]
        return {"bytes": m * d * (2 * (1 + case["adds"]) + 2 + 1) + 2 * d + 4 * m, "flops": m * d * (6 + case["adds"])}
    if case["op"] == "rows":
        return {"bytes": m * case["cols"] * 3 + 4 * m, "flops": 3 * m * case["cols"]}
    k = case["k"]
    if case["op"] == "linear":
        n = case["n"]
        return {"bytes": (m + n) * (k + 4) + 2 * m * n * (1 + case["addend"]) + 2 * n * case["bias"], "flops": 2 * m * n * k}
    n = 2 * case["inter"]
    return {"bytes": (m + n) * (k + 4) + m * n, "flops": 2 * m * n * k}


# ---- inputs ---------------------------------------------------------------------------------------------------------------------
def _codes(rows, cols):
    """Room for codes: rows start at multiples of 16 bytes, as the framework keeps them."""
    return torch.empty(rows, -(-cols // 16) * 16, dtype=_E4M3, device="cuda")[:, :cols]


def _quantise(x):
    """Codes and scales of rows, as an earlier call has left them, or as weights are stored."""
    top = x.abs().amax(-1).clamp_(min=_SMALLEST)
    codes = _codes(*x.shape)
    codes.copy_(x.mul_((_LARGEST / top).unsqueeze(-1)).clamp_(-_LARGEST, _LARGEST))
    return codes, top / _LARGEST


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, m = _TYPES[case["dtype"]], case["rows"]

    def normal(*shape, dtype=torch.float32):
        return torch.randn(shape, device="cuda", generator=g, dtype=dtype)

    def channels(n, spread):
        return torch.exp(spread * normal(n))

    s = {"case": case}
    if case["op"] == "norm":
        d = case["dim"]
        size = channels(d, 0.7)  # a residual has channels that are larger than the others throughout
        s["residual"] = (3.0 * normal(m, d) * size).to(dtype)
        s["adds"] = [(normal(m, d) * size).to(dtype) for _ in range(case["adds"])]
        s["weight"] = (0.5 * channels(d, 0.4)).to(dtype)
        s["residual_out"] = torch.empty_like(s["residual"])
        s["out"] = _codes(m, d), torch.empty(m, device="cuda")
    elif case["op"] == "rows":
        n = case["cols"]
        s["x"] = (normal(m, n + case["apart"]) * channels(n + case["apart"], 0.8)).to(dtype)[:, :n]
        s["out"] = _codes(m, n), torch.empty(m, device="cuda")
    else:
        k = case["k"]
        n = case["n"] if case["op"] == "linear" else 2 * case["inter"]
        s["x"] = _quantise(normal(m, k) * channels(k, 0.6))
        s["w"] = _quantise(normal(n, k) * (k ** -0.5 * channels(n, 0.2)).unsqueeze(-1))
        if case["op"] == "linear":
            s["bias"] = (0.3 * normal(n)).to(dtype) if case["bias"] else None
            s["addend"] = normal(m, n, dtype=dtype) if case["addend"] else None
            s["out"] = torch.empty(m, n, dtype=dtype, device="cuda")
        else:
            s["out"] = torch.empty(m, n // 2, dtype=dtype, device="cuda")
    if own:
        package = os.path.abspath("ladder-residual-inference_b200")
        if package not in sys.path:
            sys.path.insert(0, package)
        from gpt_fast import e4m3
        s["e4m3"] = e4m3
    return s


# ---- the passes -------------------------------------------------------------------------------------------------------------------
def run(s):
    case = s["case"]
    if own:
        e4m3 = s["e4m3"]
        if case["op"] == "norm":
            add1, add2 = (s["adds"] + [None, None])[:2]
            codes, scale = e4m3.add_rmsnorm(s["residual"], s["weight"], _EPS, add1=add1, add2=add2, residual_scale=case["factor"],
                                            residual_out=s["residual_out"], out=s["out"])
            return {"residual": s["residual_out"], "codes": codes, "scale": scale}
        if case["op"] == "rows":
            codes, scale = e4m3.quantize_rows(s["x"], out=s["out"])
            return {"codes": codes, "scale": scale}
        if case["op"] == "linear":
            act = None if case["act"] == "none" else case["act"]
            return e4m3.linear(s["x"], s["w"], bias=s["bias"], activation=act, addend=s["addend"], out=s["out"])
        glu = case["alpha"], float(case["limit"]), case["offset"]
        return e4m3.gateup_glu(s["x"], s["w"], glu=glu, out=s["out"])
    return {"norm": _plain_norm, "rows": _plain_rows, "linear": _plain_linear, "gateup": _plain_gateup}[case["op"]](s)


def _plain_codes(x, out):
    """x in fp32: codes against the largest magnitude of each row, which is returned."""
    top = x.abs().amax(-1).clamp(min=_SMALLEST)
    out.copy_((x * (_LARGEST / top).unsqueeze(-1)).clamp(-_LARGEST, _LARGEST))
    return top


def _plain_norm(s):
    case, dtype = s["case"], s["residual"].dtype
    x = s["residual"].float()
    if case["factor"] != 1.0:
        x = (x * case["factor"]).to(dtype).float()
    for add in s["adds"]:  # the residual is kept in its type, so each of the sums is rounded to it
        x = (x + add.float()).to(dtype).float()
    s["residual_out"].copy_(x)
    codes, scale = s["out"]
    top = _plain_codes(x * s["weight"].float(), codes)
    scale.copy_(top * torch.rsqrt((x * x).mean(-1) + _EPS) / _LARGEST)
    return {"residual": s["residual_out"], "codes": codes, "scale": scale}


def _plain_rows(s):
    codes, scale = s["out"]
    scale.copy_(_plain_codes(s["x"].float(), codes) / _LARGEST)
    return {"codes": codes, "scale": scale}


def _plain_sums(s):
    x, w = s["x"], s["w"]
    return (x[0].float() @ w[0].float().t()) * x[1].unsqueeze(-1) * w[1]


def _plain_linear(s):
    y = _plain_sums(s)
    if s["bias"] is not None:
        y = y + s["bias"].float()
    act = s["case"]["act"]
    if act == "silu":
        y = y / (1.0 + torch.exp(-y))
    elif act == "gelu":
        y = 0.5 * y * (1.0 + torch.erf(y * 0.5 ** 0.5))
    elif act == "gelu_tanh":
        y = 0.5 * y * (1.0 + torch.tanh((2.0 / math.pi) ** 0.5 * (y + 0.044715 * y * y * y)))
    if s["addend"] is not None:
        y = y + s["addend"].float()
    return s["out"].copy_(y)


def _plain_gateup(s):
    case = s["case"]
    limit = float(case["limit"])
    up, gate = _plain_sums(s).chunk(2, -1)
    gate, up = gate.clamp(max=limit), up.clamp(-limit, limit)
    return s["out"].copy_(gate / (1.0 + torch.exp(-case["alpha"] * gate)) * (up + case["offset"]))


# ---- from the definition, in 64 bits ------------------------------------------------------------------------------------------------
def _nearest_e4m3(y):
    """y, |y| <= 448, at the nearest number of three mantissa bits, ties to even; steps of 2^-9 below 2^-6."""
    _, e = torch.frexp(y)
    step = torch.exp2((e.double() - 4).clamp(min=-9))
    return torch.round(y / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rows":
        x = s["x"].double()
        top = x.abs().max(-1).values.clamp(min=_SMALLEST)
        return {"codes": _nearest_e4m3(x / top[:, None] * _LARGEST), "scale": top / _LARGEST}
    if case["op"] == "norm":
        dtype = s["residual"].dtype
        kept = s["residual"].double()
        if case["factor"] != 1.0:
            kept = (case["factor"] * kept).to(dtype).double()
        for add in s["adds"]:
            kept = kept.add_(add).to(dtype).double()
        weighted = kept * s["weight"].double()
        top = weighted.abs().max(-1).values.clamp(min=_SMALLEST)
        rms = torch.sqrt(kept.square().sum(-1) / case["dim"] + _EPS)
        return {"residual": kept, "codes": _nearest_e4m3(weighted / top[:, None] * _LARGEST), "scale": top / (rms * _LARGEST)}
    x, w = (codes.double().mul_(scale.double().unsqueeze(1)) for codes, scale in (s["x"], s["w"]))
    if case["op"] == "gateup":
        inter, limit = case["inter"], float(case["limit"])
        up = torch.einsum("mk,nk->mn", x, w[:inter]).clip(-limit, limit)
        gate = torch.einsum("mk,nk->mn", x, w[inter:]).clip(max=limit)
        return torch.sigmoid(case["alpha"] * gate).mul_(gate).mul_(up.add_(case["offset"]))
    z = torch.einsum("mk,nk->mn", x, w)
    if s["bias"] is not None:
        z += s["bias"].double()
    if case["act"] == "silu":
        z *= torch.sigmoid(z)
    elif case["act"] == "gelu":
        z = z * torch.erfc(-z / math.sqrt(2)) / 2
    elif case["act"] == "gelu_tanh":
        z = z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    return z if s["addend"] is None else z + s["addend"].double()
