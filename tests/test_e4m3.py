"""Projections in 8 bits: the host's checks of arguments, and the refusals of the C entry points, on the CPU."""
import ctypes
import math

import pytest
import torch

from e4m3_util import E4M3
from gpt_fast import _C, e4m3

BF16, FP16 = torch.bfloat16, torch.float16


def _rows(n, k):
    codes, scale = e4m3.empty_rows(n, k)
    return codes.copy_(torch.ones(n, k)), scale.fill_(1.0)


@pytest.mark.parametrize("n,k,pitch", [(1, 8, 16), (3, 16, 16), (3, 24, 32), (5, 4096, 4096), (0, 40, 48)])
def test_room_for_rows(n, k, pitch):
    codes, scale = e4m3.empty_rows(n, k)
    assert codes.dtype is E4M3 and codes.shape == (n, k) and codes.stride() == (pitch, 1) and scale.shape == (n,) and scale.dtype is torch.float32


@pytest.mark.parametrize("x", [torch.zeros(4, 12, dtype=BF16), torch.zeros(4, 16), torch.zeros(4, 4, 16, dtype=BF16), torch.zeros(4, 65544, dtype=FP16), torch.zeros(16, 4, dtype=BF16).t(),
                               torch.zeros(4, 20, dtype=BF16)[:, :16], torch.zeros(4, 0, dtype=BF16), torch.zeros(1, 16, dtype=BF16).expand(4, 16)])
def test_rows_that_are_refused(x):
    with pytest.raises(ValueError, match="^x:"):
        e4m3.quantize_rows(x)


@pytest.mark.parametrize("out", [(torch.zeros(4, 24, dtype=E4M3), torch.zeros(4)), (torch.zeros(4, 24, dtype=torch.uint8), torch.zeros(4)), (_rows(4, 24)[0], torch.zeros(5)),
                                 (_rows(4, 24)[0], torch.zeros(4, dtype=torch.float64)), (_rows(4, 24)[0], torch.zeros(8)[::2]), _rows(4, 32), _rows(5, 24)])
def test_results_that_are_refused(out):
    """Among them rows of 24 codes one behind the other, which do not start at multiples of 16 bytes."""
    with pytest.raises(ValueError, match="^out:"):
        e4m3.quantize_rows(torch.zeros(4, 24, dtype=BF16), out=out)
    with pytest.raises(ValueError, match="^out:"):
        e4m3.add_rmsnorm(torch.zeros(4, 24, dtype=BF16), torch.ones(24, dtype=BF16), 1e-5, out=out)


def test_norm_arguments():
    r, w = torch.zeros(3, 64, dtype=FP16), torch.ones(64, dtype=FP16)
    for bad in (torch.zeros(3, 64), torch.zeros(3, 60, dtype=FP16), torch.zeros(3, 16392, dtype=FP16), torch.zeros(3, 128, dtype=FP16)[:, :64]):
        with pytest.raises(ValueError, match="^residual:"):
            e4m3.add_rmsnorm(bad, w, 1e-5)
    with pytest.raises(ValueError, match="^weight:"):
        e4m3.add_rmsnorm(r, w.float(), 1e-5)
    for name in ("add1", "add2", "residual_out"):
        for bad in (torch.zeros(3, 64), torch.zeros(2, 64, dtype=FP16), torch.zeros(64, 3, dtype=FP16).t()):
            with pytest.raises(ValueError, match=f"^{name}:"):
                e4m3.add_rmsnorm(r, w, 1e-5, **{name: bad})


def test_linear_arguments():
    x, w = _rows(3, 64), _rows(10, 64)
    with pytest.raises(ValueError, match="times weights"):
        e4m3.linear(x, _rows(10, 72))
    with pytest.raises(ValueError, match="^w:"):
        e4m3.linear(x, (torch.zeros(10, 64, dtype=BF16), w[1]))
    with pytest.raises(ValueError, match="^x:"):
        e4m3.linear((x[0], x[1][:2]), w)
    with pytest.raises(ValueError, match="activation"):
        e4m3.linear(x, w, activation="tanh")
    with pytest.raises(TypeError, match="bfloat16 or float16"):
        e4m3.linear(x, w, dtype=torch.float32)
    with pytest.raises(TypeError, match="bfloat16 or float16"):
        e4m3.linear(x, w, out=torch.zeros(3, 10))
    with pytest.raises(ValueError, match="^out:"):
        e4m3.linear(x, w, out=torch.zeros(3, 12, dtype=BF16)[:, :10])
    with pytest.raises(ValueError, match="^bias:"):
        e4m3.linear(x, w, bias=torch.zeros(10))
    with pytest.raises(ValueError, match="^addend:"):
        e4m3.linear(x, w, addend=torch.zeros(3, 10, dtype=BF16), dtype=FP16)
    with pytest.raises(ValueError, match="up | gate"):
        e4m3.gateup_glu(x, _rows(9, 64))
    for limit in (-1.0, math.nan):
        with pytest.raises(ValueError, match="limit"):
            e4m3.gateup_glu(x, w, (1.0, limit, 0.0))


def test_tensors_of_the_host_are_refused():
    x, w = _rows(3, 64), _rows(10, 64)
    for call in (lambda: e4m3.quantize_rows(torch.zeros(3, 64, dtype=BF16)), lambda: e4m3.linear(x, w), lambda: e4m3.gateup_glu(x, w),
                 lambda: e4m3.add_rmsnorm(torch.zeros(3, 64, dtype=BF16), torch.ones(64, dtype=BF16), 1e-5)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


# ---- the C entry points: what they refuse never reaches a GPU ----------------------------------------------------------------------
_AT = 1 << 20  # some aligned address


def _refused(entry, packed, text):
    assert getattr(_C.lib, entry)(packed) < 0
    assert text in _C.lib.lri_last_error().decode(), _C.lib.lri_last_error()


def _quantize(x=_AT, codes=2 * _AT, scale=3 * _AT, rows=4, x_ld=64, codes_ld=64, dtype=0, cols=64):
    return _C.QUANTIZE_CALL.pack(x, codes, scale, 0, rows, x_ld, codes_ld, dtype, cols, 0)


def _norm(residual=_AT, add1=0, add2=0, weight=2 * _AT, kept=0, codes=3 * _AT, scale=4 * _AT, rows=4, codes_ld=64, dtype=0, dim=64):
    return _C.NORM8_CALL.pack(residual, add1, add2, weight, kept, codes, scale, 0, rows, codes_ld, dtype, dim, 0, 1.0, 1e-5)


def _linear(x=_AT, w=2 * _AT, xs=3 * _AT, ws=4 * _AT, bias=0, addend=0, y=5 * _AT, rows=4, x_ld=64, w_ld=64, dtype=0, n=16, k=64, act=0, limit=7.0):
    return _C.LINEAR8_CALL.pack(x, w, xs, ws, bias, addend, y, 0, rows, x_ld, w_ld, dtype, n, k, act, 1.0, limit, 0.0)


@pytest.mark.parametrize("change,text", [(dict(dtype=2), "dtype"), (dict(rows=-1), "rows"), (dict(cols=60), "multiple of 8"), (dict(cols=65544, x_ld=65544, codes_ld=65552), "65536"),
                                         (dict(codes=0), "NULL"), (dict(scale=0), "NULL"), (dict(x=0), "NULL"), (dict(codes_ld=72), "16 bytes"), (dict(codes_ld=48), "16 bytes"),
                                         (dict(codes=2 * _AT + 8), "16 bytes"), (dict(x=_AT + 8), "16 bytes"), (dict(x_ld=68), "16 bytes"), (dict(x_ld=56), "16 bytes"),
                                         (dict(scale=3 * _AT + 2), "4-byte"), (dict(codes=_AT + 16), "overlap"), (dict(scale=2 * _AT + 200), "overlap"), (dict(scale=_AT), "overlap")])
def test_quantize_refuses(change, text):
    _refused("lri_quantize_rows_e4m3", _quantize(**change), text)


@pytest.mark.parametrize("change,text", [(dict(dtype=3), "dtype"), (dict(dim=16392, codes_ld=16400), "16384"), (dict(residual=0), "NULL"), (dict(weight=0), "NULL"),
                                         (dict(add2=_AT + 4), "aligned"), (dict(kept=_AT + 16), "overlaps an input"), (dict(add1=5 * _AT, kept=5 * _AT + 32), "overlaps an input"),
                                         (dict(codes=_AT), "overlap"), (dict(kept=3 * _AT), "overlap"), (dict(kept=2 * _AT), "overlap"), (dict(scale=3 * _AT), "overlap"),
                                         (dict(add1=4 * _AT), "overlap")])
def test_norm_refuses(change, text):
    _refused("lri_add_rmsnorm_e4m3", _norm(**change), text)


@pytest.mark.parametrize("change,text", [(dict(dtype=2), "dtype"), (dict(act=5), "activation"), (dict(act=-1), "activation"), (dict(rows=-1), "rows"), (dict(n=0), "n=0"), (dict(k=60), "multiple of 8"),
                                         (dict(k=0), "multiple of 8"), (dict(act=4, bias=6 * _AT), "no bias"), (dict(act=4, addend=6 * _AT), "no bias"), (dict(act=4, limit=-1.0), "limit"),
                                         (dict(act=4, limit=math.nan), "limit"), (dict(x=0), "NULL"), (dict(ws=0), "NULL"), (dict(y=0), "NULL"), (dict(x_ld=72), "16 bytes"),
                                         (dict(w_ld=48), "16 bytes"), (dict(w=2 * _AT + 4), "16 bytes"), (dict(y=5 * _AT + 2), "aligned"), (dict(y=_AT + 32), "overlaps an input"),
                                         (dict(y=4 * _AT), "overlaps an input"), (dict(bias=5 * _AT), "overlaps an input"), (dict(addend=5 * _AT + 32), "addend that it is not")])
def test_linear_refuses(change, text):
    _refused("lri_linear_e4m3", _linear(**change), text)


@pytest.mark.parametrize("entry", ["lri_quantize_rows_e4m3", "lri_add_rmsnorm_e4m3", "lri_linear_e4m3"])
def test_no_call_and_no_rows(entry):
    _refused(entry, None, "NULL call")
    none = {"lri_quantize_rows_e4m3": _quantize(x=0, codes=0, scale=0, rows=0), "lri_add_rmsnorm_e4m3": _norm(residual=0, weight=0, codes=0, scale=0, rows=0),
            "lri_linear_e4m3": _linear(x=0, w=0, xs=0, ws=0, y=0, rows=0)}[entry]
    assert getattr(_C.lib, entry)(none) == 0


def test_structs_have_the_sizes_of_the_header():
    assert _C.QUANTIZE_CALL.size == 72 and _C.NORM8_CALL.size == 104 and _C.LINEAR8_CALL.size == 120
    assert ctypes.sizeof(ctypes.c_void_p) == 8


@pytest.mark.parametrize("change,text", [(dict(dtype=2), "dtype"), (dict(B=-1), "B=-1"), (dict(head_dim=12), "multiple of 8"), (dict(smax=0), "smax"), (dict(qkv=0), "qkv"),
                                         (dict(qkv=_AT + 8), "qkv"), (dict(table=0), "NULL"), (dict(k=3 * _AT + 4), "aligned")])
def test_rotation_refuses(change, text):
    a = dict(dtype=0, qkv=_AT, table=2 * _AT, pos=3 * _AT + 64, q=4 * _AT, k=5 * _AT, v=6 * _AT, B=1, S=2, n_head=4, n_kv=2, head_dim=64, smax=32, rows=32)
    a.update(change)
    status = _C.lib.lri_rope_kvcache(a["dtype"], a["qkv"], a["table"], a["pos"], 0, a["q"], a["k"], a["v"], a["B"], a["S"], a["n_head"], a["n_kv"], a["head_dim"], a["smax"], a["rows"], 0, None)
    assert status < 0 and text in _C.lib.lri_last_error().decode(), _C.lib.lri_last_error()
