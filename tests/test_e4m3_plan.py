"""Which kernel a projection in 8 bits takes: by rows, depth and width, and by what the caller or the process says.  On the CPU, where the library counts on 148 SMs."""
import contextlib

import pytest
import torch

from e4m3_util import check, glu64, linear64, random_rows
from gpt_fast import _C, e4m3

BF16, GLU = 0, _C.ACT_GLU


@contextlib.contextmanager
def option(name, value, default):
    _C.check(_C.lib.lri_set_option(name, value))
    try:
        yield
    finally:
        _C.check(_C.lib.lri_set_option(name, default))


def gemm_pair(value):
    return option(b"gemm_pair", value, 1)


def plan(rows, n, k, activation=0, flags=0):
    return _C.lib.lri_linear_e4m3_plan(BF16 | flags, rows, n, k, activation)


def test_which_projections_take_pairs():
    assert plan(64, 4096, 4096) == 0 and plan(4096, 8192, 8192) == 256 and plan(4096, 14336, 4096, GLU) == 256
    assert plan(1000, 2048, 8192) == 128 and plan(512, 6144, 4096) % 32 == 0 < plan(512, 6144, 4096)
    assert plan(128, 4096, 14336) == 0 < plan(128, 14336, 4096, GLU)


@pytest.mark.parametrize("activation", [0, GLU])
@pytest.mark.parametrize("k,pairs", [(8, False), (128, False), (256, False), (264, True), (1024, True)])
def test_sums_of_one_or_two_steps_stay_off_pairs(k, pairs, activation):
    assert (plan(4096, 8192, k, activation) > 0) == pairs
    with gemm_pair(256):
        assert (plan(4096, 8192, k, activation) > 0) == pairs


def test_off_pairs_by_flag_and_by_option():
    assert plan(4096, 8192, 8192, flags=_C.ONE_SM) == 0
    with gemm_pair(0):
        assert plan(4096, 8192, 8192) == plan(4096, 8192, 4096, GLU) == 0


def test_forced_on_pairs():
    with gemm_pair(96):
        assert plan(65, 100, 512) == 96 and plan(65, 100, 512, GLU) == 64 and plan(64, 100, 512) == 0 and plan(300, 100, 512, flags=_C.ONE_SM) == 0


def test_tiles_are_chosen_for_the_pairs_that_are_left():
    """64 tiles of 256 x 128 take 42 pairs two rounds, 40 of 256 x 224 one."""
    assert plan(1000, 2048, 8192) == 128
    with option(b"gemm_reserve_sms", 64, 0):
        assert plan(1000, 2048, 8192) == 224


@pytest.mark.parametrize("rows", [64 * 65535, 64 * 65535 + 1, 2 ** 31 - 300, 2 ** 31 - 1])
def test_the_most_rows(rows):
    assert plan(rows, 1, 8) == 0 and plan(rows, 8192, 8192) == 256


def test_refusals():
    for bad, text in ((dict(rows=-1), "rows"), (dict(rows=2 ** 31), "rows"), (dict(n=0), "n=0"), (dict(k=12), "multiple of 8"), (dict(activation=5), "activation"),
                      (dict(flags=2), "dtype"), (dict(flags=0x200), "dtype")):
        assert plan(**{**dict(rows=1, n=8, k=8), **bad}) < 0 and text in _C.lib.lri_last_error().decode()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n,k,kind", [(64, 1024, 1024, "linear"), (300, 4096, 1024, "linear"), (300, 1024, 256, "linear"), (2048, 1024, 264, "linear"), (300, 4096, 1024, "gateup"),
                                           (1000, 2048, 256, "gateup")])
@pytest.mark.parametrize("how", ["", "flag", "option"])
def test_kernels_follow_the_plan(rows, n, k, kind, how):
    x, w = random_rows(rows, k, 1), random_rows(n, k, 2, size=k ** -0.5)
    expected = plan(rows, n // 2 if kind == "gateup" else n, k, GLU if kind == "gateup" else 0) if not how else 0
    call = (lambda **kw: e4m3.gateup_glu(x, w, **kw)) if kind == "gateup" else (lambda **kw: e4m3.linear(x, w, **kw))
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as prof:
        with gemm_pair(0 if how == "option" else 1):
            y = call(one_sm=how == "flag")
        torch.cuda.synchronize()
    names = [e.name for e in prof.events() if "e4m3_" in e.name and e.device_type == torch.autograd.DeviceType.CUDA]
    assert len(names) == 1 and ("e4m3_pair" in names[0]) == (expected > 0), names
    if kind == "linear":
        check(y, *linear64(x, w))


@pytest.mark.gpu
def test_many_rows_off_pairs():
    """More rows than a grid's second extent has tiles, in the middle and at the end of its third."""
    rows = 2 * 64 * 65535 + 70
    few, w = random_rows(4096, 272, 1), random_rows(8, 272, 2)
    raw = few[0].view(torch.uint8)
    codes, scale = e4m3.empty_rows(rows, 272, "cuda")
    for start in range(0, rows, 4096):
        n = min(4096, rows - start)
        codes.view(torch.uint8)[start:start + n] = raw[:n]
        scale[start:start + n] = few[1][:n]
    y = e4m3.linear((codes, scale), w, one_sm=True)
    want = e4m3.linear(few, w, one_sm=True)
    check(want, *linear64(few, w))
    whole = rows // 4096 * 4096
    assert (y[:whole].view(-1, 4096, 8) == want).all() and torch.equal(y[whole:], want[:rows - whole])


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n,k,glu", [(1000, 2048, 1024, False), (600, 1500, 520, True), (300, 4096, 1024, False)])
def test_fewer_pairs(rows, n, k, glu):
    """The same results whatever is left of the chip: more rounds of tiles of other widths."""
    x, w = random_rows(rows, k, 1), random_rows(2 * n if glu else n, k, 2, size=k ** -0.5)
    call = (lambda: e4m3.gateup_glu(x, w)) if glu else (lambda: e4m3.linear(x, w))
    want = call()
    check(want, *(glu64(x, w, e4m3.SWIGLU) if glu else linear64(x, w)))
    for reserved in (1, 20, 63, 64):
        with option(b"gemm_reserve_sms", reserved, 0):
            assert torch.equal(call(), want)
