"""The kernel on pairs of SMs for projections in 8 bits: every epilogue in several rounds of tiles, so that accumulators change hands and fetching crosses tiles.  Each test asserts that
its calls take that kernel."""
import math

import pytest
import torch

from e4m3_util import check, glu64, linear64, random_rows
import gpt_fast
from gpt_fast import _C, e4m3
from paged_util import table_for
from test_paged_model import FAMILIES, PAGE, SHAPE

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16]
GLUS = [(1.0, math.inf, 0.0), (1.702, 7.0, 1.0), (1.0, 0.5, 0.0)]


def _on_pairs(rows, n, k, activation=0, rounds=1):
    """Whether a projection takes pairs, in more rounds of tiles than `rounds` (on the 74 pairs of a B200)."""
    width = _C.lib.lri_linear_e4m3_plan(0, rows, n, k, activation)
    cols = width // 2 if activation == _C.ACT_GLU else width
    return width > 0 and -(-rows // 256) * -(-n // cols) > 74 * rounds


def _guarded(rows, n, dtype):
    room = torch.full((rows + 1, n), 5.0, dtype=dtype, device="cuda")
    return room, room[:rows]


# two and three rounds; widths that are and are not multiples of 8, of 32 and of a tile; a last tile of one row and of one column
SHAPES = [(2048, 4100, 1024), (1500, 9001, 392), (1500, 9000, 392), (1300, 4001, 1160), (1025, 12008, 520)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("activation", [None, "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("bias,addend", [(False, "none"), (True, "none"), (False, "own"), (True, "own"), (True, "in place"), (False, "in place")])
@pytest.mark.parametrize("rows,n,k", SHAPES)
def test_what_follows_the_sums(dtype, activation, bias, addend, rows, n, k):
    assert _on_pairs(rows, n, k)
    x, w = random_rows(rows, k, 1, pad=rows % 2), random_rows(n, k, 2, pad=n % 3, size=2 * k ** -0.5)
    g = torch.Generator(device="cuda").manual_seed(3)
    b = (2 * torch.randn(n, generator=g, device="cuda")).to(dtype) if bias else None
    a = None if addend == "none" else torch.randn(rows, n, generator=g, device="cuda").to(dtype)
    want = linear64(x, w, b, activation, a, dtype)
    room, out = _guarded(rows, n, dtype)
    if addend == "in place":
        out.copy_(a)
        a = out
    y = e4m3.linear(x, w, bias=b, activation=activation, addend=a, out=out)
    check(y, *want)
    assert (room[rows:] == 5).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("glu", GLUS)
@pytest.mark.parametrize("rows,inter,k", [(2000, 2049, 640), (1500, 4504, 392), (1300, 2001, 1160), (1100, 3333, 264), (257, 9000, 520)])
def test_gated_unit(dtype, glu, rows, inter, k):
    assert _on_pairs(rows, inter, k, _C.ACT_GLU)
    x, w = random_rows(rows, k, 1), random_rows(2 * inter, k, 2, size=2 * k ** -0.5)
    room, out = _guarded(rows, inter, dtype)
    h = e4m3.gateup_glu(x, w, glu, out=out)
    check(h, *glu64(x, w, glu, dtype))
    assert (room[rows:] == 5).all()


def test_four_rounds():
    x, w = random_rows(4100, 264, 1), random_rows(4104, 264, 2, size=1 / 16)
    assert _on_pairs(4100, 4104, 264, rounds=3)
    y = e4m3.linear(x, w)
    check(y, *linear64(x, w))
    for _ in range(5):
        assert torch.equal(e4m3.linear(x, w), y)



@pytest.mark.parametrize("kind", ["linear", "gateup"])
def test_rows_that_are_nan_stay_alone(kind):
    rows, n, k = (1300, 4004, 1160)
    assert _on_pairs(rows, n, k) and _on_pairs(rows, n // 2, k, _C.ACT_GLU)
    x, w = random_rows(rows, k, 1), random_rows(n, k, 2, size=k ** -0.5)
    x[1][[0, 129, 1299]] = math.nan
    w[0].view(torch.uint8)[7, 9] = 0x7F
    w[1][4001] = math.nan
    y = e4m3.linear(x, w, activation="silu") if kind == "linear" else e4m3.gateup_glu(x, w, (1.0, 7.0, 0.0))
    bad = torch.zeros(rows, n, dtype=torch.bool, device="cuda")
    bad[[0, 129, 1299]], bad[:, 7], bad[:, 4001] = True, True, True
    if kind == "gateup":
        bad = bad[:, :n // 2] | bad[:, n // 2:]
    assert torch.equal(y.isnan(), bad)


def test_captured_and_without_dependent_launches():
    """A run of the operators in a graph, replayed with other inputs in place, and with kernels that do not start early."""
    rows, d, inter = 1300, 1160, 4008
    assert _on_pairs(rows, inter, d, _C.ACT_GLU) and _on_pairs(rows, d, inter, rounds=0)
    g = torch.Generator(device="cuda").manual_seed(5)
    r, a = (torch.zeros(rows, d, dtype=torch.float16, device="cuda") for _ in range(2))
    wt = torch.ones(d, dtype=torch.float16, device="cuda")
    w1, w2 = random_rows(2 * inter, d, 1, size=d ** -0.5), random_rows(d, inter, 2, size=inter ** -0.5)

    def run():
        kept = torch.empty_like(r)
        x = e4m3.add_rmsnorm(r, wt, 1e-5, a, residual_out=kept, early=True)
        h = e4m3.gateup_glu(x, w1, dtype=torch.float16)
        return e4m3.linear(e4m3.quantize_rows(h, early=True), w2, addend=kept, out=kept)

    run()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        y = run()
    for _ in range(4):
        r.copy_(torch.randn(rows, d, generator=g, device="cuda"))
        a.copy_(torch.randn(rows, d, generator=g, device="cuda"))
        graph.replay()
        assert torch.equal(y, run())
    _C.check(_C.lib.lri_set_option(b"pdl", 0))
    try:
        assert torch.equal(y, run())
    finally:
        _C.check(_C.lib.lri_set_option(b"pdl", 1))


@pytest.mark.parametrize("lo,hi", [(0, 4001), (3, 4004), (197, 4198)])
def test_parts_of_weights_and_rows(lo, hi):
    """Scales and biases that start anywhere."""
    rows, k = 1300, 1160
    assert _on_pairs(rows, hi - lo, k)
    x, w = random_rows(rows + 9, k, 1), random_rows(4200, k, 2, pad=1, size=k ** -0.5)
    bias = torch.randn(4200, dtype=torch.bfloat16, device="cuda")
    part, few = (w[0][lo:hi], w[1][lo:hi]), (x[0][5:5 + rows], x[1][5:5 + rows])
    check(e4m3.linear(few, part, bias=bias[lo:hi]), *linear64(few, part, bias[lo:hi]))


def test_every_input_may_be_a_result():
    """Rows, weights, biases and addends that the call in front has just computed."""
    rows, n, k = 1304, 1304, 1304
    assert _on_pairs(rows, n, k, rounds=0)
    x, w = random_rows(rows, k, 1), random_rows(n, k, 2, size=k ** -0.5)
    first = e4m3.linear(x, w)
    f8 = e4m3.quantize_rows(first)
    torch.cuda.synchronize()
    want = [e4m3.linear(x, w, bias=first[0], addend=first), e4m3.linear(f8, w), e4m3.linear(x, f8)]
    torch.cuda.synchronize()
    for _ in range(10):
        y, rows8 = torch.full_like(first, math.nan), e4m3.empty_rows(rows, n, "cuda")
        rows8[1].fill_(math.nan)
        e4m3.linear(x, w, out=y)
        got = [e4m3.linear(x, w, bias=y[0], addend=y)]
        e4m3.quantize_rows(y, out=rows8, early=True)
        got.append(e4m3.linear(rows8, w))
        rows8[1].fill_(math.nan)
        e4m3.quantize_rows(y, out=rows8, early=True)
        got.append(e4m3.linear(x, rows8))
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("family", list(FAMILIES))
@pytest.mark.parametrize("paged", [False, True])
def test_prompts_of_models(family, paged, monkeypatch):
    """A prompt of 2000 tokens whose projections all take pairs, each call of them against 64 bits; the same logits a second time, and a step behind it."""
    from gpt_fast.ops import CudaOps
    seen = []

    class Checked(CudaOps):
        @staticmethod
        def linear_e4m3(x, w, out, rows, n, k, x_ld, w_ld, bias=None, addend=None, activation=0, glu=(0.0, 0.0, 0.0)):
            CudaOps.linear_e4m3(x, w, out, rows, n, k, x_ld, w_ld, bias, addend, activation, glu)
            seen.append((rows, _C.lib.lri_linear_e4m3_plan(0, rows, n, k, activation) > 0))
            x = x[0][:rows], x[1][:rows]
            want = glu64(x, tuple(w), glu) if activation else linear64(x, tuple(w), addend=None if addend is None else addend.view(-1, n)[:rows])
            check(out.view(-1, n)[:rows], *want)

    mod, cls = FAMILIES[family]
    monkeypatch.setitem(mod.transformer_configs, "pairs-test", dict(SHAPE, block_size=2100, n_layer=2, n_head=8, n_local_heads=4, dim=1024, intermediate_size=2048))
    with torch.no_grad():
        with torch.device("meta"):
            model = cls.from_name("pairs-test")
        model = model.to(dtype=torch.bfloat16).to_empty(device="cuda").eval()
        g = torch.Generator(device="cuda").manual_seed(1)
        for name, p in model.named_parameters():
            p.data.copy_(torch.randn(p.shape, generator=g, device="cuda") * (0.1 if "norm" in name else p.shape[-1] ** -0.5) + (1.0 if "norm" in name else 0.0))
        model.quantize_projections()
        tokens = torch.randint(0, SHAPE["vocab_size"], (1, 2001), generator=torch.Generator().manual_seed(2)).cuda()
        pos = torch.arange(2001, dtype=torch.int32, device="cuda")
        if paged:
            pages, n_pages = table_for([2001], PAGE, device="cuda")
            model.setup_paged_caches(1, n_pages, PAGE, max_length=2048, max_prompt=2000)
            more = (pages,)
        else:
            model.setup_caches(1, 2048)
            more = ()

        def run():
            return torch.cat([model(tokens[:, :2000], pos[:2000], *more)[0], model(tokens[:, 2000:], pos[2000:], *more)[0]])
        plain = run()
        model._engine.ops = Checked
        got = run()
    assert gpt_fast._C.lib.lri_gemm_status() == 0
    assert torch.equal(got, plain) and torch.isfinite(got).all()
    assert [on for rows, on in seen if rows == 2000] == [True] * (len(seen) // 2) and not any(on for rows, on in seen if rows == 1)
