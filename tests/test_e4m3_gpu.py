"""The operators of projections in 8 bits against their definitions in 64 bits."""
import math

import pytest
import torch

from e4m3_util import E4M3, U, check, glu64, linear64, quantised, random_rows, step, values

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def e4m3():
    from gpt_fast import e4m3
    return e4m3


def _raw(codes):
    return codes.view(torch.uint8)


def _poisoned(e4m3, rows, cols, pad=0):
    """Rows for results: what lies between and behind them must stay as it is."""
    room = torch.full((rows + 2, (-(-cols // 16) + pad) * 16), 0x55, dtype=torch.uint8, device="cuda")
    scale = torch.full((rows + 2,), -3.0, device="cuda")
    return room, scale, (room.view(E4M3)[:rows, :cols], scale[:rows])


def _untouched(room, scale, rows, cols):
    assert (room[rows:] == 0x55).all() and (room[:rows, cols:] == 0x55).all() and (scale[rows:] == -3).all()


# ---- rows ------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,apart,pad", [(1, 8, 0, 0), (3, 24, 8, 1), (2, 2048, 0, 0), (149, 2056, 0, 0), (5, 4096, 1024, 0), (400, 4096, 0, 2), (2, 4104, 0, 0),
                                                 (200, 8200, 8, 0), (3, 8200, 0, 0), (150, 11000, 0, 0), (2, 16392, 0, 1), (3, 32768, 0, 0), (2, 65536, 0, 0), (160, 288, 40, 0), (150, 8, 0, 0), (151, 2040, 0, 1), (150, 30000, 0, 0), (149, 40000, 8, 0)])
def test_rows(e4m3, dtype, rows, cols, apart, pad):
    g = torch.Generator().manual_seed(rows + cols)
    wide = torch.randn(rows, cols + apart, generator=g) * torch.exp(2 * torch.randn(rows, 1, generator=g))
    wide[:, cols:] = math.nan
    x = wide.to(dtype).cuda()[:, :cols]
    room, scale, out = _poisoned(e4m3, rows, cols, pad)
    codes, got = e4m3.quantize_rows(x, out=out)
    assert codes is out[0] and got is out[1]
    want, want_scale = quantised(x)
    assert torch.equal(_raw(codes), _raw(want)) and torch.equal(got, want_scale)
    _untouched(room, scale, rows, cols)
    # and by the definition in 64 bits: the nearest code, to two roundings of the factor and one of the product
    y = x.double() / x.double().abs().amax(-1, keepdim=True) * 448
    assert ((codes.double() - y).abs() <= step(y) / 2 + 3 * U * y.abs() + 1e-30).all()
    fresh = e4m3.quantize_rows(x)
    assert torch.equal(_raw(fresh[0]), _raw(want)) and torch.equal(fresh[1], want_scale)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_no_and_of_unusual_values(e4m3, dtype):
    x = torch.randn(9, 4096).to(dtype)
    x[1] = 0.0
    x[2] = 0.0
    x[2, 77] = -0.0
    x[3] *= torch.finfo(dtype).tiny
    x[4, 4095] = math.inf
    x[5, 0] = -math.inf
    x[6, 123] = math.nan
    x[7, 5] = torch.finfo(dtype).max
    x[8] = torch.finfo(dtype).min
    x = x.cuda()
    codes, scale = e4m3.quantize_rows(x)
    want, want_scale = quantised(x)
    assert torch.equal(_raw(codes), _raw(want))
    assert torch.equal(scale.isnan(), want_scale.isnan()) and torch.equal(scale.nan_to_num(), want_scale.nan_to_num())
    assert scale.isnan().tolist() == [False] * 4 + [True] * 3 + [False] * 2
    assert (values((codes, scale))[1] == 0).all()


# ---- norm ------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,dim,adds,factor,keep", [(1, 8, 0, 1.0, "none"), (1, 4096, 1, 1.0, "own"), (7, 288, 2, 0.5, "in place"), (148, 2048, 1, 1.0, "in place"),
                                                       (149, 2304, 1, 0.125, "own"), (3, 4104, 2, 1.0, "own"), (200, 4096, 2, 1.0, "add1"), (33, 8192, 0, 1.0, "none"),
                                                       (150, 8192, 1, 1.0, "own"), (151, 11000, 1, 1.0, "own"), (2, 16384, 2, 0.25, "own"), (155, 16384, 1, 1.0, "own"), (150, 8, 1, 1.0, "in place"),
                                                       (200, 768, 2, 1.0, "own"), (149, 2040, 0, 1.0, "none"), (160, 5120, 2, 1.0, "in place")])
def test_norm(e4m3, dtype, rows, dim, adds, factor, keep):
    from gpt_fast.ops import CudaOps
    g = torch.Generator().manual_seed(rows * dim)
    residual = (torch.randn(rows, dim, generator=g) * torch.exp(torch.randn(dim, generator=g)) * 3).to(dtype).cuda()
    added = [torch.randn(rows, dim, generator=g).to(dtype).cuda() for _ in range(adds)] + [None] * (2 - adds)
    weight = torch.randn(dim, generator=g).to(dtype).cuda()
    eps = 1e-5
    # the residual, bit for bit as the operator of 16 bits leaves it
    kept, normed = torch.empty_like(residual), torch.empty_like(residual)
    CudaOps.add_rmsnorm(residual, *added, weight, eps, kept, normed, rows, factor)
    x = kept.double()
    room, scale, out = _poisoned(e4m3, rows, dim)
    to = {"none": None, "own": torch.full_like(residual, 7.0), "in place": residual, "add1": added[0]}[keep]
    codes, got = e4m3.add_rmsnorm(residual, weight, eps, *added, residual_scale=factor, residual_out=to, out=out)
    if to is not None:
        assert torch.equal(to, kept)
    want, top = quantised(kept.float() * weight.float())  # (the product is exact)
    assert torch.equal(_raw(codes), _raw(want))
    _untouched(room, scale, rows, dim)
    rms = (x.square().mean(-1) + eps).sqrt()
    exact = (x * weight.double()).abs().amax(-1) / (448 * rms)
    # the sum of squares: at most 64 terms a thread, 10 levels of joining, half of it in the root; rsqrtf to 2 ulp, five more roundings
    assert ((got.double() - exact).abs() <= (37 + 4 + 5) * U * exact).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_norm_of_unusual_rows(e4m3, dtype):
    residual = torch.randn(6, 512).to(dtype)
    add = torch.randn(6, 512).to(dtype)
    residual[1], add[1] = 0.0, 0.0
    residual[2, 3] = math.inf
    add[3, 511] = math.nan
    residual[4], add[4] = torch.finfo(dtype).tiny, 0.0
    residual[5, 0], add[5, 0] = math.inf, -math.inf
    residual, add, weight = residual.cuda(), add.cuda(), torch.randn(512).to(dtype).cuda()
    codes, scale = e4m3.add_rmsnorm(residual, weight, 1e-6, add)
    assert scale.isnan().tolist() == [False, False, True, True, False, True]
    assert (_raw(codes)[2] == 0).all() and (values((codes, scale))[1] == 0).all()
    want, _ = quantised((residual + add).float() * weight.float())
    assert torch.equal(_raw(codes), _raw(want))
    assert torch.isfinite(scale[[0, 1, 4]]).all()


# ---- linear ----------------------------------------------------------------------------------------------------------------------
SIZES = [(1, 8), (8, 8), (17, 24), (130, 136), (100, 1000), (2001, 264), (256, 4096), (1280, 2048), (4096, 1024), (640, 11000), (129, 16384)]


@pytest.mark.parametrize("n,k", SIZES)
@pytest.mark.parametrize("rows", [1, 2, 7, 8, 9, 16, 17, 33, 64, 65, 127, 128, 129, 200, 257, 384, 1000])
def test_linear(e4m3, rows, n, k):
    dtype = TYPES[(rows + n) % 2]
    x, w = random_rows(rows, k, rows + k, pad=rows % 3), random_rows(n, k, n, pad=n % 2, size=k ** -0.5)
    room = torch.full((rows + 1, n), 5.0, dtype=dtype, device="cuda")
    y = e4m3.linear(x, w, out=room[:rows])
    check(y, *linear64(x, w, dtype=dtype))
    assert (room[rows:] == 5).all()
    assert torch.equal(y, e4m3.linear(x, w, dtype=dtype)), "the same call twice"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("activation", [None, "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("bias,addend", [(True, "none"), (False, "own"), (True, "in place")])
@pytest.mark.parametrize("rows,n,k", [(1, 520, 264), (5, 333, 1000), (40, 1056, 512), (100, 257, 128), (300, 520, 640), (513, 203, 72)])
def test_what_follows_the_sums(e4m3, dtype, activation, bias, addend, rows, n, k):
    x, w = random_rows(rows, k, 1), random_rows(n, k, 2, size=2 * k ** -0.5)
    g = torch.Generator().manual_seed(3)
    b = (2 * torch.randn(n, generator=g)).to(dtype).cuda() if bias else None
    a = None if addend == "none" else torch.randn(rows, n, generator=g).to(dtype).cuda()
    want = linear64(x, w, b, activation, a, dtype)
    y = e4m3.linear(x, w, bias=b, activation=activation, addend=a, dtype=dtype, out=a if addend == "in place" else None)
    check(y, *want)


GLUS = [(1.0, math.inf, 0.0), (1.702, 7.0, 1.0), (1.0, 0.5, 0.0)]


@pytest.mark.parametrize("rows", [1, 3, 8, 9, 16, 33, 64, 65, 128, 129, 300, 520])
@pytest.mark.parametrize("inter,k,glu", [(1, 8, GLUS[0]), (60, 136, GLUS[1]), (129, 1000, GLUS[0]), (1024, 2048, GLUS[2]), (2001, 264, GLUS[1]), (500, 11000, GLUS[0])])
def test_gateup(e4m3, rows, inter, k, glu):
    dtype = TYPES[(rows + inter) % 2]
    x, w = random_rows(rows, k, rows), random_rows(2 * inter, k, inter, size=2 * k ** -0.5)
    room = torch.full((rows + 1, inter), 5.0, dtype=dtype, device="cuda")
    h = e4m3.gateup_glu(x, w, glu, out=room[:rows])
    check(h, *glu64(x, w, glu, dtype))
    assert (room[rows:] == 5).all()


@pytest.mark.parametrize("rows,n,k", [(257, 640, 11000), (256, 4096, 14336), (300, 1333, 8200), (1000, 1001, 12296), (512, 4096, 9000), (131, 2048, 16384), (1024, 200, 5000)])
@pytest.mark.parametrize("how", ["plain", "all"])
def test_few_tiles_of_long_sums(e4m3, rows, n, k, how):
    """Few tiles, many steps each: the ends of the rounds of both kernels."""
    dtype = TYPES[n % 2]
    x, w = random_rows(rows, k, 1), random_rows(n, k, 2, size=2 * k ** -0.5)
    g = torch.Generator().manual_seed(3)
    more = {} if how == "plain" else dict(bias=torch.randn(n, generator=g).to(dtype).cuda(), activation="gelu", addend=torch.randn(rows, n, generator=g).to(dtype).cuda())
    room = torch.full((rows + 1, n), 5.0, dtype=dtype, device="cuda")
    y = e4m3.linear(x, w, out=room[:rows], **more)
    check(y, *linear64(x, w, dtype=dtype, **more))
    assert (room[rows:] == 5).all()
    for _ in range(5):
        assert torch.equal(y, e4m3.linear(x, w, dtype=dtype, **more))


@pytest.mark.parametrize("rows,inter,k", [(1000, 1024, 8192), (257, 1500, 6000), (512, 2047, 9000), (1024, 130, 4104)])
@pytest.mark.parametrize("glu", GLUS)
def test_gateup_of_few_tiles_and_long_sums(e4m3, rows, inter, k, glu):
    dtype = TYPES[inter % 2]
    x, w = random_rows(rows, k, 1), random_rows(2 * inter, k, 2, size=2 * k ** -0.5)
    h = e4m3.gateup_glu(x, w, glu, dtype=dtype)
    check(h, *glu64(x, w, glu, dtype))
    for _ in range(5):
        assert torch.equal(h, e4m3.gateup_glu(x, w, glu, dtype=dtype))


@pytest.mark.parametrize("rows", [2, 20, 100, 300])
@pytest.mark.parametrize("kind", ["linear", "gateup"])
def test_rows_that_are_nan_stay_alone(e4m3, rows, kind):
    """A NaN scale makes its row NaN, a NaN code of a weight its output; an infinite limit lets NaN through."""
    x, w = random_rows(rows, 256, 1), random_rows(200, 256, 2, size=1 / 16)
    x[1][1] = math.nan
    _raw(w[0])[7, 9] = 0x7F
    w[1][150] = math.nan
    y = e4m3.linear(x, w) if kind == "linear" else e4m3.gateup_glu(x, w, (1.0, 7.0, 0.0))
    bad = torch.zeros(rows, 200, dtype=torch.bool, device="cuda")
    bad[1], bad[:, 7], bad[:, 150] = True, True, True
    if kind == "gateup":
        bad = bad[:, :100] | bad[:, 100:]
    assert torch.equal(y.isnan(), bad)


@pytest.mark.parametrize("rows", [1, 30, 100, 400])
def test_zero_rows_and_zero_weights(e4m3, rows):
    x, w = random_rows(rows, 512, 1), random_rows(96, 512, 2)
    _raw(x[0])[0] = 0
    x[1][0] = 0.0
    assert (e4m3.linear(x, w)[0] == 0).all()
    none = e4m3.linear((x[0][:0], x[1][:0]), w)
    assert none.shape == (0, 96)


@pytest.mark.parametrize("rows", [1, 40, 300])
def test_weights_of_the_call_before(e4m3, rows):
    """A projection starts on its weights before the kernel in front of it is complete; the rows that the operators store may be weights all the same."""
    x = random_rows(rows, 4096, 1)
    w = torch.randn(512, 4096, dtype=torch.bfloat16, device="cuda")
    add = torch.randn_like(w)
    ones = torch.ones(4096, dtype=torch.bfloat16, device="cuda")
    codes, scale = e4m3.empty_rows(512, 4096, "cuda")
    for turn in range(20):
        _raw(codes).fill_(0x7F)
        scale.fill_(math.nan)
        if turn % 2:
            e4m3.quantize_rows(w, out=(codes, scale))
        else:
            e4m3.add_rmsnorm(w, ones, 1e-5, add1=add, out=(codes, scale))
        y = e4m3.linear(x, (codes, scale))
        check(y, *linear64(x, (codes, scale)))


# ---- calls around calls ------------------------------------------------------------------------------------------------------------
SHAPES = [(1, 640, 1024, False), (40, 1100, 512, True), (100, 300, 2048, False), (300, 1100, 512, True), (700, 512, 264, False)]


def _call(e4m3, rows, n, k, glu, seed=0):
    x, w = random_rows(rows, k, seed), random_rows(n, k, seed + 1, size=2 * k ** -0.5)
    return (lambda: e4m3.gateup_glu(x, w, GLUS[1])) if glu else (lambda: e4m3.linear(x, w, activation="silu"))


def test_two_streams_at_once(e4m3):
    """Calls share nothing on the device."""
    calls = [_call(e4m3, *s, seed=i) for i, s in enumerate(SHAPES)]
    want = [c() for c in calls]
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for turn in range(20):
        for i, c in enumerate(calls):
            with torch.cuda.stream(streams[(i + turn) % 3]):
                got.append((i, c()))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i, y in got)


@pytest.mark.parametrize("rows", [3, 90, 400])
def test_captured(e4m3, rows):
    """A run of the operators in a graph, replayed with other inputs in place."""
    d, inter = 512, 1000
    g = torch.Generator().manual_seed(5)
    r, a, wt = torch.zeros(rows, d, dtype=torch.float16, device="cuda"), torch.zeros(rows, d, dtype=torch.float16, device="cuda"), torch.ones(d, dtype=torch.float16, device="cuda")
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
        r.copy_(torch.randn(rows, d, generator=g))
        a.copy_(torch.randn(rows, d, generator=g))
        graph.replay()
        assert torch.equal(y, run())


def test_without_dependent_launches(e4m3):
    from gpt_fast import _C
    calls = [_call(e4m3, *s, seed=i) for i, s in enumerate(SHAPES)]
    x = torch.randn(50, 2048, dtype=torch.float16, device="cuda")
    want, rows = [c() for c in calls], e4m3.quantize_rows(x)
    _C.check(_C.lib.lri_set_option(b"pdl", 0))
    try:
        assert all(torch.equal(c(), w) for c, w in zip(calls, want))
        assert torch.equal(_raw(e4m3.quantize_rows(x)[0]), _raw(rows[0]))
    finally:
        _C.check(_C.lib.lri_set_option(b"pdl", 1))


@pytest.mark.parametrize("rows", [1, 20, 300])
@pytest.mark.parametrize("lo,hi", [(0, 7), (3, 200), (197, 333)])
def test_parts_of_weights_and_rows(e4m3, rows, lo, hi):
    """Rows lo .. hi of a weight and of activations: scales and biases that start anywhere."""
    x, w = random_rows(rows + 9, 264, 1), random_rows(333, 264, 2, pad=1)
    bias = torch.randn(333, dtype=torch.bfloat16, device="cuda")
    part = w[0][lo:hi], w[1][lo:hi]
    few = x[0][5:5 + rows], x[1][5:5 + rows]
    check(e4m3.linear(few, part, bias=bias[lo:hi]), *linear64(few, part, bias[lo:hi]))
    if (hi - lo) % 2 == 0:
        check(e4m3.gateup_glu(few, part), *glu64(few, part, GLUS[0]))


def test_many_rows(e4m3):
    """More rows than a grid's second extent has tiles."""
    x, w = random_rows(64 * 65535 + 70, 16, 1), random_rows(8, 16, 2)
    y = e4m3.linear(x, w)
    at = torch.cat([torch.arange(300), torch.arange(x[0].shape[0] - 300, x[0].shape[0])]).cuda()
    check(y[at], *linear64((x[0][at], x[1][at]), w))
    assert torch.equal(y[:128], e4m3.linear((x[0][:128], x[1][:128]), w))


def test_another_device_is_refused(e4m3):
    x, w = random_rows(3, 64, 1), random_rows(8, 64, 2)
    with pytest.raises(RuntimeError, match="no CPU path"):
        e4m3.linear(x, (w[0], w[1].cpu()))
    with pytest.raises(RuntimeError, match="no CPU path"):
        e4m3.quantize_rows(torch.zeros(3, 64, dtype=torch.bfloat16, device="cuda"), out=e4m3.empty_rows(3, 64, "cpu"))


def test_addends_and_biases_of_the_call_before(e4m3):
    """Only weights are read ahead: what a call has just computed may be the next one's bias or addend."""
    x, w = random_rows(1, 2048, 1), random_rows(2048, 2048, 2, size=2048 ** -0.5)
    first = e4m3.linear(x, w)
    torch.cuda.synchronize()
    want = e4m3.linear(x, w, bias=first[0], addend=first)
    for _ in range(20):
        y = torch.full_like(first, math.nan)
        e4m3.linear(x, w, out=y)
        assert torch.equal(e4m3.linear(x, w, bias=y[0], addend=y), want)
