"""Models on paged caches: prompts of unequal lengths one after the other, whole and in portions, then steps of all sequences together, against the same
model on dense caches with each sequence alone.  On the CPU with stand-in operators (the schedules), on the GPU with the kernels."""
import pytest
import torch

import gpt_fast
from gpt_fast import gpt_dense_TP, gpt_desync_TP, gpt_ladder_TP, gpt_parallel_TP
from paged_ops import PagedOps
from paged_util import E4M3, table_for

FAMILIES = {"dense": (gpt_dense_TP, gpt_fast.GPTDense), "ladder": (gpt_ladder_TP, gpt_fast.GPTLadder),
            "parallel": (gpt_parallel_TP, gpt_fast.GPTParallel), "desync": (gpt_desync_TP, gpt_fast.GPTDesync)}
SHAPE = dict(block_size=256, vocab_size=512, n_layer=3, n_head=4, n_local_heads=2, dim=256, intermediate_size=512, rope_base=500000)
PROMPTS, STEPS, PAGE = [70, 1, 33], 4, 16


def _model(family, device, seed=0):
    mod, cls = FAMILIES[family]
    mod.transformer_configs["paged-test"] = dict(SHAPE)
    with torch.device("meta"):
        model = cls.from_name("paged-test")
    model = model.to(dtype=torch.bfloat16).to_empty(device=device).eval()
    g = torch.Generator().manual_seed(seed)
    for name, p in model.named_parameters():
        scale = 1.0 if "norm" in name or "embeddings" in name else p.shape[-1] ** -0.5
        p.data.copy_((torch.randn(p.shape, generator=g) * (0.1 if "norm" in name else scale) + (1.0 if "norm" in name else 0.0)).to(p.dtype))
    return model


def _run_paged(model, tokens, device, cache_dtype, portion=None, patch=lambda m: None):
    pages, n_pages = table_for([n + STEPS for n in PROMPTS], PAGE, device=device)
    model.setup_paged_caches(len(PROMPTS) + 1, n_pages, PAGE, max_length=128, max_prompt=96, cache_dtype=cache_dtype)
    patch(model)
    out = [[] for _ in PROMPTS]
    for b, n in enumerate(PROMPTS):
        for at in range(0, n, portion or n):
            end = min(n, at + (portion or n))
            logits = model(tokens[b][None, at:end].to(device), torch.arange(at, end, dtype=torch.int32, device=device), pages[b:b + 1])
            out[b].append(logits[0].float().cpu())
    # an idle row among the live ones
    rows = [0, 1, None, 2]
    table = torch.full((4, pages.shape[1]), -1, dtype=torch.int32, device=device)
    for r, b in enumerate(rows):
        if b is not None:
            table[r] = pages[b]
    for s in range(STEPS):
        idx = torch.tensor([[0 if b is None else tokens[b][PROMPTS[b] + s]] for b in rows], device=device)
        pos = torch.tensor([-1 if b is None else PROMPTS[b] + s for b in rows], dtype=torch.int32, device=device)
        logits = model(idx, pos, table)
        for r, b in enumerate(rows):
            if b is not None:
                out[b].append(logits[r].float().cpu())
    return [torch.cat(o) for o in out]


def _run_dense(model, tokens, device, patch=lambda m: None):
    out = []
    for b, n in enumerate(PROMPTS):
        model.setup_caches(1, 128)
        patch(model)
        o = [model(tokens[b][None, :n].to(device), torch.arange(n, dtype=torch.int32, device=device))[0].float().cpu()]
        for s in range(STEPS):
            o.append(model(tokens[b][None, n + s:n + s + 1].to(device), torch.tensor([n + s], dtype=torch.int32, device=device))[0].float().cpu())
        out.append(torch.cat(o))
    return out


def _tokens():
    return torch.randint(0, SHAPE["vocab_size"], (len(PROMPTS), max(PROMPTS) + STEPS), generator=torch.Generator().manual_seed(7))


def _cpu(model):
    from cpu_ops import CpuOps

    class Ops(PagedOps, CpuOps):
        pass

    model._engine.ops = Ops
    for layer in model.layers:
        layer.attention.kv_cache.ops = Ops


@pytest.fixture
def no_library(monkeypatch):
    """Set-up asks the library for sizes only; on the CPU its workspaces are empty."""
    from gpt_fast.paged import PagedKVCache
    monkeypatch.setattr(PagedKVCache, "ops", PagedOps)


@pytest.mark.parametrize("family", list(FAMILIES))
@pytest.mark.parametrize("portion", [None, 32])
def test_schedules_on_the_cpu(family, portion, no_library):
    with torch.no_grad():
        model, tokens = _model(family, "cpu"), _tokens()
        want = _run_dense(model, tokens, "cpu", _cpu)
        got = _run_paged(model, tokens, "cpu", None, portion, _cpu)
    # both in bf16 with the same roundings: sums differ in the last place of 32 bits at most, which may turn a rounding now and then
    for g, w in zip(got, want):
        assert ((g - w).norm() / w.norm()).item() < 1e-2


def test_what_is_refused(no_library):
    model = _model("dense", "cpu")
    with pytest.raises(AssertionError):
        model(torch.zeros(1, 1, dtype=torch.long), torch.zeros(1, dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32))
    with pytest.raises(AssertionError):
        model.setup_paged_caches(2, 8, 16, max_length=512)
    model.setup_paged_caches(2, 8, 16, max_length=64, max_prompt=32)
    _cpu(model)
    zeros, pages = torch.zeros(4, dtype=torch.int32), torch.zeros(2, 4, dtype=torch.int32)
    for idx, pos, table in ((torch.zeros(1, 1), zeros[:1], None), (torch.zeros(2, 2), zeros, pages), (torch.zeros(2, 1), zeros[:1], pages),
                            (torch.zeros(1, 4), zeros, pages), (torch.zeros(3, 1), zeros[:3], pages), (torch.zeros(1, 33), torch.zeros(33, dtype=torch.int32), pages[:1])):
        with pytest.raises(AssertionError):
            model(idx.long(), pos, table)
    model.setup_caches(2, 32)
    _cpu(model)
    assert model(torch.zeros(2, 3, dtype=torch.long), torch.arange(3)).shape == (2, 3, SHAPE["vocab_size"])
    with pytest.raises(AssertionError):
        model(torch.zeros(2, 1, dtype=torch.long), zeros[:2], pages)


def test_layer_lists_keep_their_own_caches():
    with torch.device("meta"):
        model = gpt_fast.GPTPatevik.from_name("patevik-tiny")
    with pytest.raises(TypeError):
        model.setup_paged_caches(1, 8)


# whole models against one another: the tolerance of the other whole-model tests
TOL = 2e-2


@pytest.mark.gpu
@pytest.mark.parametrize("family", list(FAMILIES))
@pytest.mark.parametrize("portion", [None, 32])
def test_pages_against_dense_caches(family, portion):
    with torch.no_grad():
        model, tokens = _model(family, "cuda"), _tokens()
        want = _run_dense(model, tokens, "cuda")
        got = _run_paged(model, tokens, "cuda", None, portion)
    for g, w in zip(got, want):
        assert ((g - w).norm() / w.norm()).item() < TOL


@pytest.mark.gpu
@pytest.mark.parametrize("family", ["dense", "parallel"])
def test_e4m3_pages_against_plain_operators(family):
    """The same model with the cache's kernels and with plain torch in their place."""
    def plain(model):
        for layer in model.layers:
            layer.attention.kv_cache.ops = PagedOps

    with torch.no_grad():
        model, tokens = _model(family, "cuda"), _tokens()
        got = _run_paged(model, tokens, "cuda", E4M3)
        want = _run_paged(model, tokens, "cuda", E4M3, patch=plain)
    for g, w in zip(got, want):
        assert ((g - w).norm() / w.norm()).item() < TOL


@pytest.mark.gpu
@pytest.mark.parametrize("family", ["ladder", "dense"])
def test_captured_steps(family):
    """A step captured once and replayed while tokens and positions change in place and an idle row comes to life; the greedy head; the sampled one."""
    with torch.no_grad():
        model, tokens = _model(family, "cuda"), _tokens()
        pages, n_pages = table_for([n + STEPS for n in PROMPTS], PAGE)
        model.setup_paged_caches(3, n_pages, PAGE, max_length=128, max_prompt=96)

        def prompts():
            return [model.prefill_last(tokens[b][None, :n].cuda(), torch.arange(n, dtype=torch.int32, device="cuda"), pages[b:b + 1]) for b, n in enumerate(PROMPTS)]

        prompts()
        idx, pos = torch.zeros(3, 1, dtype=torch.int32, device="cuda"), torch.full((3,), -1, dtype=torch.int32, device="cuda")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            model(idx, pos, pages)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            logits = model(idx, pos, pages)
        for s in range(STEPS):
            now = [PROMPTS[0] + s, PROMPTS[1] + s if s else -1, PROMPTS[2] + s]
            pos.copy_(torch.tensor(now, dtype=torch.int32))
            idx.copy_(torch.stack([tokens[b][PROMPTS[b] + s] for b in range(3)])[:, None])
            graph.replay()
            got = logits.clone()
            want = model(idx, pos, pages)  # the same step again writes the same rows
            live = [b for b in range(3) if now[b] >= 0]
            assert torch.equal(got[live], want[live])
            top = want[live, -1].float().topk(2).values
            decided = (top[:, 0] - top[:, 1]) > TOL * want[live, -1].float().abs().amax(-1)
            chosen = model.decode_greedy(idx, pos, pages)[live, 0].long()
            assert (chosen == want[live, -1].argmax(-1))[decided].all()
            drawn = model.decode_sample(idx, pos, top_k=1, pages=pages)[live, 0].long()
            assert (drawn == want[live, -1].argmax(-1))[decided].all()


@pytest.mark.gpu
def test_trace_names_the_paged_operators():
    """The per-operation times of a step and of a prompt hold what the layers' caches call; afterwards the caches call the library itself again."""
    from gpt_fast.ops import CudaOps
    from gpt_fast.trace import trace_engine
    with torch.no_grad():
        model, tokens = _model("ladder", "cuda"), _tokens()
        pages, n_pages = table_for([PROMPTS[0] + STEPS], PAGE)
        model.setup_paged_caches(1, n_pages, PAGE, max_length=128, max_prompt=96)
        n, layers = PROMPTS[0], len(model.layers)
        trace = trace_engine(model._engine)
        model.prefill_last(tokens[0][None, :n].cuda(), torch.arange(n, dtype=torch.int32, device="cuda"), pages)
        model(tokens[0][None, n:n + 1].cuda(), torch.tensor([n], dtype=torch.int32, device="cuda"), pages)
        report = trace.report()
        trace.stop()
        assert report["rope_paged_store"][0] == 2 * layers and report["paged_attention"][0] == report["paged_load"][0] == layers
        assert all(layer.attention.kv_cache.ops is CudaOps for layer in model.layers)
