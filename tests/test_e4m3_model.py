"""Models whose projections are in 8 bits: every schedule, on dense caches and on pages, against the same arithmetic by another way; on the CPU with stand-in
operators (the schedules), on the GPU with the kernels."""
import os
import subprocess
import sys

import pytest
import torch

import gpt_fast
from e4m3_ops import E4M3Ops, fake_weights, faked_ops
from e4m3_util import check, glu64, linear64, quantised
from gpt_fast import e4m3
from paged_ops import PagedOps
from test_paged_model import FAMILIES, PROMPTS, STEPS, _model, _run_dense, _run_paged, _tokens

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _apart(got, want):
    return max(((g - w).norm() / w.norm()).item() for g, w in zip(got, want))


def _stand_in(base):
    """A model's patch: operators of 8 bits in plain torch over `base`."""
    class Ops(E4M3Ops, base):
        pass

    def patch(model):
        model._engine.ops = Ops
    return patch


def _cpu_ops():
    from cpu_ops import CpuOps

    class Ops(E4M3Ops, PagedOps, CpuOps):
        pass
    return Ops


def _on_cpu(model):
    model._engine.ops = _cpu_ops()
    for layer in model.layers:
        layer.attention.kv_cache.ops = model._engine.ops


@pytest.fixture
def no_library(monkeypatch):
    from gpt_fast.paged import PagedKVCache
    monkeypatch.setattr(PagedKVCache, "ops", PagedOps)
    monkeypatch.setattr(e4m3, "CudaOps", E4M3Ops)


@pytest.mark.parametrize("family", list(FAMILIES))
@pytest.mark.parametrize("paged", [False, True])
def test_schedules_on_the_cpu(family, paged, no_library):
    """The model in 16 bits with weights and inputs of its projections brought to 8 bits and back.  There the norm's rows are rounded to bfloat16 before (2^-9),
    which turns one code in twenty by a step of a sixteenth to an eighth, and the values are rounded after: 2 % for a projection, about as much of the
    whole.  A wrong order of adds or a buffer in use twice leaves nothing alike."""
    def faked(model):
        model._engine.ops = faked_ops(model.config.vocab_size)

    with torch.no_grad():
        tokens = _tokens()
        plain = _model(family, "cpu")
        fake_weights(plain)
        want = _run_dense(plain, tokens, "cpu", faked)
        model = _model(family, "cpu").quantize_projections()
        assert not any(isinstance(m, torch.nn.Linear) for m in model.layers.modules()) and isinstance(model.output, torch.nn.Linear)
        got = _run_paged(model, tokens, "cpu", None, None, _on_cpu) if paged else _run_dense(model, tokens, "cpu", _on_cpu)
    assert _apart(got, want) < 0.08


def test_what_is_refused(no_library):
    with pytest.raises(TypeError, match="16 bits"):
        with torch.device("meta"):
            gpt_fast.GPTPatevik.from_name("patevik-1b").quantize_projections()
    model = _model("dense", "cpu")
    model.setup_caches(1, 32)
    with pytest.raises(RuntimeError, match="before caches"):
        model.quantize_projections()
    lin = e4m3.E4M3Linear(torch.randn(24, 40, dtype=torch.bfloat16))
    assert lin.codes.shape == (24, 48) and (lin.codes.view(torch.uint8)[:, 40:] == 0).all()
    codes, scale = lin.weight[8:16]
    assert codes.data_ptr() == lin.codes[8:].data_ptr() and codes.shape == (8, 40) and scale.shape == (8,)
    again = e4m3.E4M3Linear(torch.zeros(24, 40, dtype=torch.bfloat16))
    again.load_state_dict(lin.state_dict())
    assert torch.equal(again.codes.view(torch.uint8), lin.codes.view(torch.uint8)) and torch.equal(again.scale, lin.scale)
    with pytest.raises(TypeError, match="cast"):
        lin.to(torch.float16).weight


@pytest.mark.parametrize("world", [1, 2])
def test_ranks(world):
    cmd = [sys.executable, "-m", "torch.distributed.run", "--nnodes=1", f"--nproc-per-node={world}", "--master-addr", "127.0.0.1",
           "--master-port", str(29830 + world), os.path.join(ROOT, "tests", "e4m3_cpu_worker.py")]
    r = subprocess.run(cmd, capture_output=True, text=True, timeout=600, env=dict(os.environ, OMP_NUM_THREADS="2", CUDA_VISIBLE_DEVICES=""))
    assert r.returncode == 0, r.stdout[-3000:] + r.stderr[-3000:]
    assert "E4M3-CPU-OK" in r.stdout


# ---- on the GPU --------------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("family", list(FAMILIES))
@pytest.mark.parametrize("kind", ["dense", "paged", "paged e4m3"])
def test_models(family, kind):
    """Each operator of the run against its definition, and the whole against the run with stand-ins.  There any difference grows to what roundings to 8 bits
    leave: where inputs differ by e of their size, e / s of the codes differ by a step s (a sixteenth to an eighth), that is by sqrt(e s) of the whole, which
    is more than e below s.  From sums that differ in the last place, 2^-24, three roundings lead to 2^-3 (2^-24 / 2 + 3 / 2 .. = -13.5, -8.3, -5.6 in powers of two)
    and further ones nowhere: the bound is that of roundings that have nothing to do with each other, as on the CPU."""
    from gpt_fast.ops import CudaOps
    tokens = _tokens()
    cache = torch.float8_e4m3fn if kind.endswith("e4m3") else None
    seen = []

    class Checked(CudaOps):
        @staticmethod
        def quantize_rows_e4m3(x, codes, scale, rows, *args, **kw):
            CudaOps.quantize_rows_e4m3(x, codes, scale, rows, *args, **kw)
            want, s = quantised(x[:rows])
            assert torch.equal(codes[:rows].view(torch.uint8), want.view(torch.uint8)) and torch.equal(scale[:rows], s)
            seen.append("rows")

        @staticmethod
        def add_rmsnorm_e4m3(residual, add1, add2, weight, eps, residual_out, codes, scale, rows, dim, codes_ld, residual_scale=1.0, early=False):
            x, normed = torch.empty_like(residual), torch.empty_like(residual)
            CudaOps.add_rmsnorm(residual, add1, add2, weight, eps, x, normed, rows, residual_scale)
            CudaOps.add_rmsnorm_e4m3(residual, add1, add2, weight, eps, residual_out, codes, scale, rows, dim, codes_ld, residual_scale, early)
            want, _ = quantised(x[:rows].float() * weight.float())
            assert residual_out is None or torch.equal(residual_out[:rows], x[:rows])
            assert torch.equal(codes[:rows].view(torch.uint8), want.view(torch.uint8))
            seen.append("norm")

        @staticmethod
        def linear_e4m3(x, w, out, rows, n, k, x_ld, w_ld, bias=None, addend=None, activation=0, glu=(0.0, 0.0, 0.0)):
            CudaOps.linear_e4m3(x, w, out, rows, n, k, x_ld, w_ld, bias, addend, activation, glu)
            x = x[0][:rows], x[1][:rows]
            want = glu64(x, tuple(w), glu) if activation else linear64(x, tuple(w), addend=None if addend is None else addend.view(-1, n)[:rows])
            check(out.view(-1, n)[:rows], *want)
            seen.append("glu" if activation else "linear")

    def checked(model):
        model._engine.ops = Checked

    with torch.no_grad():
        model = _model(family, "cuda").quantize_projections()

        def run(patch):
            model.max_seq_length = -1  # fresh caches
            return _run_dense(model, tokens, "cuda", patch) if kind == "dense" else _run_paged(model, tokens, "cuda", cache, 32 if cache else None, patch)
        plain = run(lambda m: None)
        got = run(checked)
        assert gpt_fast._C.lib.lri_gemm_status() == 0
        want = run(_stand_in(CudaOps))
    assert seen.count("linear") == 3 * seen.count("glu") and seen.count("rows") == 2 * seen.count("glu") > 0
    assert seen.count("norm") == seen.count("glu") * (1 if family == "parallel" else 2)
    assert all(torch.equal(p, g) for p, g in zip(plain, got))
    assert _apart(got, want) < 0.08


@pytest.mark.gpu
@pytest.mark.parametrize("family", list(FAMILIES))
@pytest.mark.parametrize("batch", [1, 5, 70])
def test_captured_steps(family, batch):
    """A step in a graph gives the bits of an eager one, and the loop on the device its tokens."""
    from gpt_fast.generate import DeviceLoop
    with torch.no_grad():
        model = _model(family, "cuda").quantize_projections()
        model.setup_caches(batch, 64)
        prompt = torch.randint(0, 512, (batch, 9), generator=torch.Generator().manual_seed(3)).cuda()
        first = model.prefill_last(prompt, torch.arange(9, dtype=torch.int32, device="cuda"))[:, -1].argmax(-1, keepdim=True)
        pos = torch.tensor([9], dtype=torch.int32, device="cuda")
        eager = model(first, pos).clone()
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            model(first, pos)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                logits = model(first, pos)
        torch.cuda.current_stream().wait_stream(stream)
        for _ in range(3):
            logits.zero_()
            graph.replay()
            assert torch.equal(logits, eager)
        if batch <= 64:
            want, token = [], first
            for s in range(6):
                token = model.decode_greedy(token, torch.tensor([9 + s], dtype=torch.int32, device="cuda")).clone()
                want.append(token)
            loop = DeviceLoop(model, batch, steps_per_replay=3)
            loop.start(first, 9)
            assert torch.equal(loop.run(6).view(batch, 6), torch.cat(want, 1).view(batch, 6))


@pytest.mark.gpu
@pytest.mark.parametrize("family", ["dense", "parallel"])
def test_layers_by_themselves(family):
    """The modules' own forward, as the reference's blocks call them."""
    with torch.no_grad():
        model = _model(family, "cuda").quantize_projections()
        model.setup_caches(2, 64)
        x = torch.randn(2, 7, 256, dtype=torch.bfloat16, device="cuda")
        pos = torch.arange(7, dtype=torch.int32, device="cuda")
        att = model.layers[0].attention
        got = att(x, model.freqs_cis[pos.long()], None, pos)
        x8 = e4m3.quantize_rows(x.view(14, 256))
        w = att.wqkv.weight if family == "dense" else att.wqkv1.weight
        n = (att.n_head + 2 * att.n_local_heads) * att.head_dim
        qkv = e4m3.linear(x8, w[:n])
        q = torch.empty(14, att.n_head * att.head_dim, dtype=torch.bfloat16, device="cuda")
        k, v = torch.zeros_like(att.kv_cache.k_cache), torch.zeros_like(att.kv_cache.v_cache)
        E4M3Ops.rope_kvcache(qkv, model.freqs_cis, False, pos, q, k, v, 2, 7, att.n_head, att.n_local_heads, att.head_dim)
        assert torch.equal(k, att.kv_cache.k_cache) and torch.equal(v, att.kv_cache.v_cache)
        y = torch.empty_like(q)
        gpt_fast.ops.CudaOps.attention(q, k, v, pos, y, 2, 7, att.n_head, att.n_local_heads, att.head_dim, None, 1)
        want = e4m3.linear(e4m3.quantize_rows(y), att.wo.weight)
        if family == "parallel":
            h = e4m3.gateup_glu(x8, w[n:])
            want = e4m3.linear(e4m3.quantize_rows(h), att.w2.weight, addend=want)
        assert torch.equal(got.view(14, 256), want)
        if family == "dense":
            ff = model.layers[0].feed_forward
            h = e4m3.gateup_glu(x8, ff.w1.weight)
            assert torch.equal(ff(x).view(14, 256), e4m3.linear(e4m3.quantize_rows(h), ff.w2.weight))


@pytest.mark.gpu
def test_a_run_of_the_operators():
    """A feed-forward block as a model runs it, three rows of which are of no use: adds and norm, gated unit, rows, down projection onto the residual."""
    g = torch.Generator().manual_seed(0)
    d, inter = 520, 1000
    for rows in (1, 30, 200):
        r, a = (torch.randn(rows, d, generator=g).to(torch.bfloat16).cuda() for _ in range(2))
        if rows > 3:
            r[1], a[1], r[3, 5] = 0.0, 0.0, float("nan")
        weight = torch.rand(d, generator=g).to(torch.bfloat16).cuda()
        w1, w2 = (e4m3.E4M3Linear(torch.randn(n, k, generator=g).mul(k ** -0.5).to(torch.bfloat16).cuda()) for n, k in ((2 * inter, d), (d, inter)))
        kept = torch.empty_like(r)
        x = e4m3.add_rmsnorm(r, weight, 1e-5, a, residual_out=kept, early=True)
        h = e4m3.gateup_glu(x, w1.weight)
        y = e4m3.linear(e4m3.quantize_rows(h, early=True), w2.weight, addend=kept)
        assert torch.equal(kept, r + a) or rows > 3
        v = (r + a).double()
        v = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-5) * weight.double()
        up, gate = (v @ (w1.weight.codes.double() * w1.scale.double().unsqueeze(1)).t()).chunk(2, -1)
        want = (torch.sigmoid(gate) * gate * up) @ (w2.weight.codes.double() * w2.scale.double().unsqueeze(1)).t() + (r + a).double()
        if rows > 3:
            assert y[3].isnan().all() and (y[1] == 0).all() and torch.isfinite(y[[0, 2, 4]]).all()
        live = [i for i in range(rows) if rows <= 3 or i not in (1, 3)]
        # two roundings of rows to 8 bits (at most a sixteenth, a thirtieth on the average) on the way of sums that are about half of the result
        assert ((y.double() - want)[live].norm() / want[live].norm()).item() < 0.05
