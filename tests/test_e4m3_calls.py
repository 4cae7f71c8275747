"""Calls of the operators of 8 bits that their documentation allows: on the CPU as far as the host's part goes."""
import pytest
import torch

from e4m3_util import random_rows
from gpt_fast import e4m3


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
