"""The sources of the kernels of 8-bit projections: what a warp has to do together is done by lanes that have met.  (Lanes leave a polling loop one by one; an .aligned
barrier or a load from tensor memory that they then come to one by one is undefined and can hang, so this is read, not run.)"""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ladder-residual-inference_b200", "csrc")
KERNELS = ["e4m3_few.cu", "e4m3_pair.cu"]


def _statements(name):
    """The lines of a file that are neither empty nor comments."""
    with open(os.path.join(CSRC, name)) as f:
        lines = [re.sub(r"\s*//.*", "", line).strip() for line in f]
    return [line for line in lines if line]


@pytest.mark.parametrize("name", KERNELS + ["gemm_pair.cu"])
def test_cluster_barriers_are_the_converging_ones(name):
    assert not [line for line in _statements(name) if "barrier.cluster" in line]


def test_cluster_barriers_converge():
    lines = _statements("cluster.cuh")
    at = [i for i, line in enumerate(lines) if "barrier.cluster" in line]
    assert len(at) == 3 and all(lines[i - 1] == "__syncwarp();" for i in at)


@pytest.mark.parametrize("name", KERNELS)
def test_loads_from_tensor_memory_converge(name):
    """Behind a __syncwarp, with nothing in between but declarations and branches that a whole warp takes alike."""
    lines = _statements(name)
    at = [i for i, line in enumerate(lines) if "tmem_ld" in line]
    assert at
    for i in at:
        before = [line for line in lines[i - 3:i] if line not in ("uint32_t r[32];", "if (kGlu) {")]
        assert before[-1] == "__syncwarp();", lines[i - 3:i + 1]
