"""Ladder models some of whose layers are dense, with their projections in 8 bits: the schedule with two pending addends."""
import pytest
import torch

from e4m3_ops import fake_weights, faked_ops
from test_e4m3_model import _apart, _on_cpu, _stand_in, no_library  # noqa: F401
from test_paged_model import SHAPE, _model, _run_dense, _run_paged, _tokens

MIXES = [[0], [0, 2]]


@pytest.mark.parametrize("layers", MIXES)
@pytest.mark.parametrize("paged", [False, True])
def test_schedules_on_the_cpu(layers, paged, no_library, monkeypatch):  # noqa: F811
    """The bound of test_e4m3_model.test_schedules_on_the_cpu, for the reasons that stand there."""
    monkeypatch.setitem(SHAPE, "ladder_layers", layers)

    def faked(model):
        model._engine.ops = faked_ops(model.config.vocab_size)

    with torch.no_grad():
        tokens = _tokens()
        plain = _model("ladder", "cpu")
        fake_weights(plain)
        want = _run_dense(plain, tokens, "cpu", faked)
        model = _model("ladder", "cpu").quantize_projections()
        assert model.config.ladder_layers == layers
        got = _run_paged(model, tokens, "cpu", None, None, _on_cpu) if paged else _run_dense(model, tokens, "cpu", _on_cpu)
    assert _apart(got, want) < 0.08


@pytest.mark.gpu
@pytest.mark.parametrize("layers", MIXES)
def test_against_stand_ins(layers, monkeypatch):
    """Kernels against operators in plain torch: the bound of roundings to 8 bits that have nothing to do with each other (test_e4m3_model.test_models)."""
    from gpt_fast.ops import CudaOps
    monkeypatch.setitem(SHAPE, "ladder_layers", layers)
    with torch.no_grad():
        model = _model("ladder", "cuda").quantize_projections()

        def run(patch):
            model.max_seq_length = -1  # fresh caches
            return _run_dense(model, _tokens(), "cuda", patch)
        got = run(lambda m: None)
        assert all(torch.equal(a, b) for a, b in zip(got, run(lambda m: None)))
        want = run(_stand_in(CudaOps))
    assert _apart(got, want) < 0.08
