"""Calls of the operators of 8 bits that their documentation allows: on the CPU as far as the host's part goes."""
import pytest
import torch

from e4m3_ops import E4M3Ops
from e4m3_util import random_rows
from gpt_fast import _C, e4m3


def test_rows_of_a_weight_as_activations():
    """A pair is a pair: also rows that a module owns."""
    w = e4m3.E4M3Weight(*random_rows(16, 64, 1, device="cpu"))
    for call in (e4m3.linear, e4m3.gateup_glu):
        with pytest.raises(RuntimeError, match="no CPU path"):  # (the last of the host's checks)
            call(w[:5], w)


@pytest.mark.gpu
def test_rows_of_a_weight_as_activations_on_the_gpu():
    w = e4m3.E4M3Weight(*random_rows(16, 64, 1))
    x = w[:5]
    assert torch.equal(e4m3.linear(x, w), e4m3.linear(tuple(x), tuple(w)))
    assert torch.equal(e4m3.gateup_glu(x, w), e4m3.gateup_glu(tuple(x), tuple(w)))


def _tiny(monkeypatch, **shape):
    from gpt_fast import gpt_dense_TP
    from test_paged_model import SHAPE
    monkeypatch.setitem(gpt_dense_TP.transformer_configs, "eight-test", {**SHAPE, **shape})
    monkeypatch.setattr(e4m3, "CudaOps", E4M3Ops)
    return gpt_dense_TP.GPTDense.from_name("eight-test").to(torch.bfloat16)


def _linears(model):
    return [type(m) for m in model.layers.modules() if isinstance(m, (torch.nn.Linear, e4m3.E4M3Linear))]


@pytest.mark.parametrize("fault", ["width", "bias", "type", "device", "address"])
def test_a_model_is_quantised_as_a_whole_or_not_at_all(fault, monkeypatch):
    """The last layer's last projection cannot go to 8 bits: the others stay as they are."""
    model = _tiny(monkeypatch, **({"intermediate_size": 516} if fault == "width" else {}))
    last = model.layers[-1].feed_forward.w2
    if fault == "bias":
        last.bias = torch.nn.Parameter(torch.zeros(256, dtype=torch.bfloat16))
    elif fault == "type":
        last.float()
    elif fault == "device":
        last.to("meta")
    elif fault == "address":
        n = last.weight.numel()
        last.weight.data = torch.zeros(n + 4, dtype=torch.bfloat16)[4:].view(last.weight.shape)
    before = _linears(model)
    with pytest.raises(ValueError):
        model.quantize_projections()
    assert _linears(model) == before and e4m3.E4M3Linear not in before


def test_quantised_twice(monkeypatch):
    model = _tiny(monkeypatch)
    assert model.quantize_projections() is model
    kept = [m.codes.data_ptr() for m in model.modules() if isinstance(m, e4m3.E4M3Linear)]
    model.quantize_projections()
    assert kept and kept == [m.codes.data_ptr() for m in model.modules() if isinstance(m, e4m3.E4M3Linear)]


@pytest.mark.parametrize("q,k,v", [(0, 1 << 21, 1 << 22), (256, 1 << 21, 1 << 22), (1 << 20, 512, 1 << 22), (1 << 20, 1 << 21, 1008)])
def test_rotation_in_place_is_refused(q, k, v):
    """Queries have another pitch than the rows that they come from: a thread would overwrite what another has yet to read."""
    at = 1 << 24
    status = _C.lib.lri_rope_kvcache(0, at, 1 << 20, 1 << 21, 0, at + q, at + k, at + v, 1, 2, 4, 2, 64, 32, 32, 0, None)
    assert status < 0 and b"overlap" in _C.lib.lri_last_error()
