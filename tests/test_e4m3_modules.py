"""The layers' own forward: what stands where a projection was is its weight, in 16 or 8 bits."""
import pytest
import torch
import torch.nn as nn

from cpu_ops import CpuOps
from e4m3_ops import E4M3Ops
from gpt_fast import e4m3, utils
from test_paged_model import _model


class _Stand(nn.Module):
    """Owns a weight as a projection does; its own forward is another program's."""

    def __init__(self, lin):
        super().__init__()
        self.weight = lin.weight

    def forward(self, x):
        raise AssertionError("the layers multiply by the weight")


class _Ops(E4M3Ops, CpuOps):
    pass


@pytest.fixture
def on_cpu(monkeypatch):
    monkeypatch.setattr(utils, "_ops", lambda: _Ops)
    monkeypatch.setattr(e4m3, "CudaOps", _Stored)


class _Stored(E4M3Ops):
    """As the kernels take their arguments: contiguous results of the sizes that are said."""

    @staticmethod
    def linear_e4m3(x, w, out, rows, n, k, x_ld, w_ld, bias=None, addend=None, activation=0, glu=(0.0, 0.0, 0.0), flags=0):
        assert out.shape == (rows, n) and tuple(w)[0].shape[1] == k
        E4M3Ops.linear_e4m3(x, w, out, rows, n, k, x_ld, w_ld, bias, addend, activation, glu)


def _names(family):
    return ("wqkv1", "wo", "w2") if family == "parallel" else ("wqkv", "wo")


def _run(model, family):
    x = torch.randn(2, 7, 256, dtype=torch.bfloat16, generator=torch.Generator().manual_seed(1))
    pos = torch.arange(7, dtype=torch.int32)
    layer = model.layers[0]
    out = [layer.attention(x, model.freqs_cis[pos.long()], None, pos)]
    if family != "parallel":
        out.append(layer.feed_forward(x))
    return out


@pytest.mark.parametrize("family", ["dense", "parallel"])
def test_other_modules_with_a_weight(family, on_cpu):
    with torch.no_grad():
        model = _model(family, "cpu")
        model.setup_caches(2, 32)
        want = _run(model, family)
        layer = model.layers[0]
        for part, names in ((layer.attention, _names(family)), (getattr(layer, "feed_forward", None), ("w1", "w2"))):
            for name in names if part is not None else ():
                setattr(part, name, _Stand(getattr(part, name)))
        got = _run(model, family)
    assert all(torch.equal(g, w) for g, w in zip(got, want))


@pytest.mark.parametrize("family", ["dense", "parallel"])
def test_layers_in_8_bits(family, on_cpu):
    """The layer's forward in 8 bits against the one in 16: two or three projections with rows and weights in 8 bits, 3 % each."""
    with torch.no_grad():
        model = _model(family, "cpu")
        model.setup_caches(2, 32)
        want = _run(model, family)
        eight = _model(family, "cpu").quantize_projections()
        eight.setup_caches(2, 32)
        got = _run(eight, family)
    for g, w in zip(got, want):
        assert ((g.float() - w.float()).norm() / w.float().norm()).item() < 0.12
