"""What a projection in 8 bits reads before the kernel in front of it on the stream is complete: its weights, where the caller says that they may be, and nothing else."""
import pytest
import torch

from e4m3_util import check, linear64, random_rows
from gpt_fast import _C, e4m3
from test_e4m3_model import _on_cpu, no_library  # noqa: F401
from test_paged_model import FAMILIES, _model, _run_dense, _tokens


def test_weights_are_read_ahead_where_it_is_said(no_library):  # noqa: F811
    lin = e4m3.E4M3Linear(torch.randn(24, 40, dtype=torch.bfloat16))
    assert not lin.weight.ahead and not lin.weight[8:].ahead
    w = e4m3.E4M3Weight(*lin.weight, ahead=True)
    assert w.ahead and w[:8].ahead and tuple(w)[0] is w.codes


@pytest.mark.parametrize("family", list(FAMILIES))
def test_the_engine_reads_its_weights_ahead(family, no_library):  # noqa: F811
    seen = []

    def patch(model):
        _on_cpu(model)
        ops = model._engine.ops

        class Recorded(ops):
            @staticmethod
            def linear_e4m3(x, w, *args, **kw):
                seen.append(w.ahead)
                ops.linear_e4m3(x, w, *args, **kw)

            @staticmethod
            def embedding(*args):
                seen.append("embedding")
                ops.embedding(*args)
        model._engine.ops = Recorded

    with torch.no_grad():
        _run_dense(_model(family, "cpu").quantize_projections(), _tokens(), "cpu", patch)
    assert seen[0] == "embedding" and True in seen and False not in seen


class _Recorder:
    """The library, with the calls of projections written down."""

    def __init__(self, lib, calls):
        self.lib, self.calls = lib, calls

    def __getattr__(self, name):
        fn = getattr(self.lib, name)
        if name != "lri_linear_e4m3":
            return fn

        def call(packed):
            self.calls.append(_C.LINEAR8_CALL.unpack(packed)[11])
            return fn(packed)
        return call


@pytest.mark.gpu
def test_flags_of_calls(monkeypatch):
    calls = []
    x, w = random_rows(3, 64, 1), random_rows(8, 64, 2)
    want = e4m3.linear(x, w)
    monkeypatch.setattr(_C, "lib", _Recorder(_C.lib, calls))
    lin = e4m3.E4M3Linear(torch.randn(16, 64, dtype=torch.bfloat16, device="cuda"))
    lin(torch.randn(2, 64, dtype=torch.bfloat16, device="cuda"))
    e4m3.gateup_glu(x, w)
    assert torch.equal(e4m3.linear(x, w), want) and calls == [0, 0, 0]
    assert torch.equal(e4m3.linear(x, e4m3.E4M3Weight(*w, ahead=True)), want) and calls[3:] == [_C.WEIGHTS_AHEAD]
    e4m3.gateup_glu(x, e4m3.E4M3Weight(*w, ahead=True), dtype=torch.float16, one_sm=True)
    assert calls[4:] == [_C.WEIGHTS_AHEAD | _C.ONE_SM | _C.FP16]


SIZES = [(1, 512, 4096), (40, 512, 4096), (300, 4096, 1024)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n,k", SIZES)
@pytest.mark.parametrize("between", [0, 1, 2])
def test_weights_that_calls_before_have_stored(rows, n, k, between):
    """Weights stored, then rows that let the next kernel start at once, then the product: as a module that is used as soon as it is made."""
    assert (_C.lib.lri_linear_e4m3_plan(0, rows, n, k, 0) > 0) == (rows == 300)
    g = torch.Generator(device="cuda").manual_seed(rows)
    weights = [torch.randn(n, k, dtype=torch.bfloat16, device="cuda", generator=g) for _ in range(2)]
    a = torch.randn(rows, k, dtype=torch.bfloat16, device="cuda", generator=g)
    want = []
    for w in weights:
        x8, w8 = e4m3.quantize_rows(a), e4m3.quantize_rows(w)
        torch.cuda.synchronize()
        want.append(e4m3.linear(x8, w8))
        check(want[-1], *linear64(x8, w8))
    x8, w8 = e4m3.empty_rows(rows, k, "cuda"), e4m3.empty_rows(n, k, "cuda")
    torch.cuda.synchronize()
    got = []
    for turn in range(40):
        e4m3.quantize_rows(weights[turn % 2], out=w8, early=True)
        for _ in range(between):
            e4m3.quantize_rows(a, out=x8, early=True)
        if between == 0 and turn == 0:
            e4m3.quantize_rows(a, out=x8)
            e4m3.quantize_rows(weights[0], out=w8, early=True)
        got.append(e4m3.linear(x8, w8))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[turn % 2]) for turn, y in enumerate(got))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,dim", [(1, 4096), (160, 512), (150, 8192)])
def test_the_weight_of_a_norm_may_be_a_result(rows, dim):
    g = torch.Generator(device="cuda").manual_seed(dim)
    r = torch.randn(rows, dim, dtype=torch.bfloat16, device="cuda", generator=g)
    x, w = random_rows(1, 512, 1), [random_rows(dim, 512, seed, size=512 ** -0.5) for seed in (2, 3)]
    out = torch.empty(1, dim, dtype=torch.bfloat16, device="cuda")
    want = []
    for v in w:
        weight = e4m3.linear(x, v)[0].clone()
        torch.cuda.synchronize()
        want.append(e4m3.add_rmsnorm(r, weight, 1e-5))
    torch.cuda.synchronize()
    got = []
    for turn in range(20):
        e4m3.linear(x, w[turn % 2], out=out)
        got.append(e4m3.add_rmsnorm(r, out[0], 1e-5, early=True))
    torch.cuda.synchronize()
    for turn, (codes, scale) in enumerate(got):
        assert torch.equal(codes.view(torch.uint8), want[turn % 2][0].view(torch.uint8)) and torch.equal(scale, want[turn % 2][1])


@pytest.mark.gpu
@pytest.mark.parametrize("dim,batch,two", [(256, 1, False), (256, 50, False), (256, 65, False), (4096, 1, False), (4096, 30, True)])
def test_streams_of_ladder_steps(dim, batch, two, monkeypatch):
    """Two streams in a graph up to 64 sequences; called eagerly only where the device takes longer than the host.  The same bits."""
    from gpt_fast.engine import Engine
    from test_paged_model import SHAPE
    if dim == 4096:
        monkeypatch.setitem(SHAPE, "dim", 4096)
        monkeypatch.setitem(SHAPE, "n_head", 32)
        monkeypatch.setitem(SHAPE, "n_local_heads", 8)
        monkeypatch.setitem(SHAPE, "intermediate_size", 14336)
        monkeypatch.setitem(SHAPE, "n_layer", 2)
    taken = []
    for name in ("_run_ladder_one_stream", "_run_ladder_two_streams"):
        def run(self, *args, _run=getattr(Engine, name), _two=name.endswith("two_streams")):
            taken.append(_two)
            _run(self, *args)
        monkeypatch.setattr(Engine, name, run)
    with torch.no_grad():
        model = _model("ladder", "cuda").quantize_projections()
        model.setup_caches(batch, 32)
        idx = torch.randint(0, 512, (batch, 1), generator=torch.Generator().manual_seed(1)).cuda()
        pos = torch.tensor([0], dtype=torch.int32, device="cuda")
        eager = model(idx, pos).clone()
        assert taken == [two]
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            logits = model(idx, pos)
        assert taken[1:] == [batch <= 64]
        graph.replay()
        assert torch.equal(logits, eager)
