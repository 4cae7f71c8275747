"""Models on pages where a token has no place of its own, or an earlier position has no page.  On the CPU with stand-in operators, on the GPU with the
kernels: `_setup` takes care of the difference."""
import pytest
import torch

from cpu_ops import CpuOps
from paged_ops import PagedOps
from test_paged_model import SHAPE, _model

PAGE = 16


class Ops(PagedOps, CpuOps):
    @staticmethod
    def _rows(stored, scales, pages, b, lo, hi):
        """As the kernels: a position behind the table's pages counts as the last of them, numbers that name no page are none."""
        n_pages, page = stored.shape[0], stored.shape[2]
        named = torch.where((pages >= 0) & (pages < n_pages), pages, -1)
        return PagedOps._rows(stored, scales, named, b, lo, min(hi, pages.shape[1] * page))

    @classmethod
    def paged_load(cls, k_pages, v_pages, k_scale, v_scale, pages, last_pos, k_out, v_out, rows, pages_shape, cache_shape):
        n_pages, _, page, _ = cache_shape
        for b, last in enumerate(last_pos.tolist()):
            n = max(0, min(last + 1, rows, pages_shape[1] * page))
            at = torch.arange(n)
            ids = pages[b].long()[at // page]
            there = (ids >= 0) & (ids < n_pages)
            for t, s, out in ((k_pages, k_scale, k_out), (v_pages, v_scale, v_out)):
                out[b, :, :-(-n // 64) * 64] = 0
                out[b][:, at[there]] = cls._rows(t, s, pages, b, 0, n).transpose(0, 1).to(out.dtype)

    @staticmethod
    def attention_pages(q, k_cache, v_cache, input_pos, pages, page, n_pages, out, S, n_head, n_kv, head_dim):
        most = min(k_cache.shape[2], pages.shape[1] * page)
        at = torch.arange(most)
        ids = pages[0].long()[at // page]
        seen = (at <= input_pos.long()[:, None]) & (ids >= 0) & (ids < n_pages)
        k, v = (t[0, :, :most].float().repeat_interleave(n_head // n_kv, 0) for t in (k_cache, v_cache))
        scores = (q.float().view(S, n_head, head_dim).transpose(0, 1) @ k.transpose(1, 2) * head_dim ** -0.5).masked_fill(~seen, float("-inf"))
        w = torch.softmax(scores, -1).nan_to_num(0.0)  # nothing visible: zeros
        out[:S] = (w @ v).transpose(0, 1).reshape(S, -1).to(out.dtype)


BOTH = [pytest.param("cpu"), pytest.param("cuda", marks=pytest.mark.gpu)]


def _setup(monkeypatch, family, device, *args, **kw):
    if device == "cpu":
        from gpt_fast.paged import PagedKVCache
        monkeypatch.setattr(PagedKVCache, "ops", Ops)
    model = _model(family, device)
    model.setup_paged_caches(*args, **kw)
    if device == "cpu":
        model._engine.ops = Ops
    return model


def _tokens(n, seed):
    return torch.randint(0, SHAPE["vocab_size"], (1, n), generator=torch.Generator().manual_seed(seed))


def _positions(at, end, device):
    return torch.arange(at, end, dtype=torch.int32, device=device)


@pytest.mark.parametrize("device", BOTH)
@pytest.mark.parametrize("family", ["dense", "ladder", "parallel"])
def test_a_step_without_its_page_depends_on_nothing_before_it(family, device, monkeypatch):
    """The newest position of a live row has no page yet, or lies behind the table: what comes back is the same bits after steps of other tokens and other
    sequences, since nothing that they left behind takes part."""
    with torch.no_grad():
        model = _setup(monkeypatch, family, device, 3, 12, PAGE, max_length=128, max_prompt=64)
        table = torch.full((3, 6), -1, dtype=torch.int32, device=device)
        table[0, :2], table[1, :3], table[2, :2] = (torch.tensor(x, dtype=torch.int32) for x in ([0, 1], [2, 3, 4], [5, 6]))
        for b, n in enumerate((32, 40, 32)):  # rows 0 and 2 fill their pages
            model(_tokens(n, b).to(device), _positions(0, n, device), table[b:b + 1])
        idx = _tokens(3, 9).t().contiguous().to(device)
        got = []
        for seed in (1, 2):
            other = torch.full_like(table, -1)
            other[:, :2] = torch.tensor([[7 + seed, 10], [10, 11], [7, 8]], dtype=torch.int32)
            model(_tokens(3, 20 + seed).t().contiguous().to(device), torch.tensor([4 + seed, 3, 2], dtype=torch.int32, device=device), other)
            # row 0: no page at its position; row 1: all there; row 2: a position behind the table
            got.append(model(idx, torch.tensor([32, 40, 6 * PAGE], dtype=torch.int32, device=device), table).float().cpu())
        assert got[0].isfinite().all() and torch.equal(got[0], got[1])


def _same(got, want):
    """The tolerance of the other whole-model tests."""
    assert got.isfinite().all() and ((got - want).norm() / want.norm()).item() < 2e-2


def _singles(model, tokens, positions, table, device):
    return torch.cat([model(tokens[:, i:i + 1].to(device), torch.tensor([p], dtype=torch.int32, device=device), table)[0].float().cpu()
                      for i, p in enumerate(positions)])


@pytest.mark.parametrize("device", BOTH)
@pytest.mark.parametrize("family", ["dense", "ladder"])
@pytest.mark.parametrize("gone", [[0, 1], [2], [5], [0, 3, 4, 5]])
def test_a_portion_sees_what_single_steps_see(family, device, gone, monkeypatch):
    """Pages of earlier positions that were freed, and pages that some of the new tokens lack: a portion of a prompt and the same tokens one at a time."""
    with torch.no_grad():
        model = _setup(monkeypatch, family, device, 1, 12, PAGE, max_length=128, max_prompt=96)
        table = torch.arange(8, dtype=torch.int32, device=device)[None].clone()
        model(_tokens(70, 1).to(device), _positions(0, 70, device), table)
        table[0, gone] = -1
        table[0, 7] = 12  # names no page either
        tokens = _tokens(40, 2)
        got = model(tokens.to(device), _positions(70, 110, device), table)[0].float().cpu()
        _same(got, _singles(model, tokens, range(70, 110), table, device))


@pytest.mark.parametrize("device", BOTH)
@pytest.mark.parametrize("family", ["dense", "ladder"])
def test_a_padded_portion(family, device, monkeypatch):
    """Tokens without a position at the end of a portion, and in it: the others' logits are those of single steps, and nothing comes from another sequence's
    prompt, whose copy lay in the same place."""
    with torch.no_grad():
        model = _setup(monkeypatch, family, device, 1, 24, PAGE, max_length=128, max_prompt=96)
        table, other = (torch.arange(8, dtype=torch.int32, device=device)[None] + i for i in (0, 12))
        model(_tokens(30, 1).to(device), _positions(0, 30, device), table)
        tokens, live = _tokens(40, 2), list(range(6)) + list(range(9, 33))
        positions = torch.full((40,), -1, dtype=torch.int32, device=device)
        positions[live] = _positions(30, 60, device)
        got = []
        for seed in (3, 4):
            model(_tokens(90, seed).to(device), _positions(0, 90, device), other)
            got.append(model(tokens.to(device), positions, table)[0].float().cpu())
        assert torch.equal(*got)
        _same(got[0][live], _singles(model, tokens[:, live], range(30, 60), table, device))
        nothing = torch.full((40,), -1, dtype=torch.int32, device=device)
        got = []
        for seed in (3, 4):
            model(_tokens(90, seed).to(device), _positions(0, 90, device), other)
            got.append(model(tokens.to(device), nothing, table)[0].float().cpu())
        assert torch.equal(*got)


@pytest.mark.parametrize("device", BOTH)
@pytest.mark.parametrize("family", ["dense", "ladder"])
def test_portions_behind_max_length(family, device, monkeypatch):
    """A table with room for more positions than max_length: portions behind it see all of the sequence, as steps do."""
    with torch.no_grad():
        model = _setup(monkeypatch, family, device, 1, 24, PAGE, max_length=64, max_prompt=64)
        table = torch.arange(24, dtype=torch.int32, device=device)[None]
        for at in (0, 50, 100, 150):
            tokens = _tokens(50, at)
            got = model(tokens.to(device), _positions(at, at + 50, device), table)[0].float().cpu()
        _same(got, _singles(model, tokens, range(150, 200), table, device))


@pytest.mark.gpu
@pytest.mark.parametrize("family", ["ladder", "dense"])
def test_captured_portions(family):
    """A portion captured once, behind a table that is wider than max_length, and replayed while tokens, positions and pages change in place; another sequence's
    prompt runs in between, and a smaller captured portion of before the copy grew still replays."""
    with torch.no_grad():
        model = _model(family, "cuda")
        model.setup_paged_caches(1, 40, PAGE, max_length=64, max_prompt=64)

        def capture(tokens, positions, table):
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                model(tokens, positions, table)
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                return graph, model(tokens, positions, table)

        calls = []
        for most, n in ((4, 20), (10, 40)):
            call = [torch.zeros(1, n, dtype=torch.int64, device="cuda"), torch.full((n,), -1, dtype=torch.int32, device="cuda"),
                    torch.full((1, most), -1, dtype=torch.int32, device="cuda")]
            calls.append((n, call) + capture(*call))
        other = torch.arange(20, 30, dtype=torch.int32, device="cuda")[None]
        for i, at in enumerate((0, 10, 24)):
            for n, call, graph, logits in calls:
                call[0].copy_(_tokens(n, i))
                call[1].copy_(_positions(at, at + n, "cuda"))
                call[1][n - i:] = -1
                call[2].copy_(torch.arange(call[2].shape[1], device="cuda").int() + i)
                if i == 2:
                    call[2][0, 0] = -1
                model(_tokens(60, 7).cuda(), _positions(90, 150, "cuda"), other)
                graph.replay()
                got = logits.clone()
                model(_tokens(60, 8).cuda(), _positions(90, 150, "cuda"), other)
                assert torch.equal(got, model(*call))  # the same portion again writes the same rows


@pytest.mark.parametrize("kw,most", [(dict(), 256), (dict(max_length=100), 100), (dict(max_length=1), 1), (dict(max_prompt=40), 40), (dict(max_length=64, max_prompt=64), 64)])
def test_the_longest_prompt(kw, most, monkeypatch):
    """By default 512 tokens, or as many as a sequence has."""
    with torch.no_grad():
        model = _setup(monkeypatch, "dense", "cpu", 1, 16, PAGE, **kw)
        table = torch.arange(16, dtype=torch.int32)[None]
        assert model(_tokens(most, 0), _positions(0, most, "cpu"), table).shape == (1, most, SHAPE["vocab_size"])
        with pytest.raises(AssertionError):
            model(_tokens(most + 1, 0), _positions(0, most + 1, "cpu"), table)


@pytest.mark.parametrize("kw,named", [(dict(max_length=257), "max_length=257"), (dict(max_length=0), "max_length=0"), (dict(max_length=64, max_prompt=65), "max_prompt=65"),
                                      (dict(max_prompt=0), "max_prompt=0")])
def test_set_up_names_what_it_refuses(kw, named, monkeypatch):
    with pytest.raises(AssertionError, match=named):
        _setup(monkeypatch, "dense", "cpu", 1, 16, PAGE, **kw)


# The C ABI checks sizes and pointers before it touches a device: addresses that are never read stand in for device memory.
BUF = 1 << 20
ARG, ALIGN, UNSUPPORTED = -1, -2, -3


@pytest.mark.parametrize("kw,status", [
    (dict(pages=0), ARG), (dict(most=0), ARG), (dict(n_pages=0), ARG), (dict(page=12), ARG), (dict(page=0), ARG), (dict(page=8192), ARG),
    (dict(most=1 << 28), ARG), (dict(q=0), ARG), (dict(pos=0), ARG), (dict(out=BUF + 8), ALIGN), (dict(S=-1), ARG), (dict(n_head=3), ARG), (dict(dim=80), UNSUPPORTED),
    (dict(smax=0), ARG), (dict(smax=72), ARG), (dict(dtype=3), UNSUPPORTED), (dict(S=0), 0)])
def test_c_prompt_over_pages_refuses(kw, status):
    from gpt_fast import _C
    a = dict(dtype=0, q=BUF, k=BUF, v=BUF, pos=BUF, i64=0, out=BUF, S=4, n_head=4, n_kv=2, dim=64, smax=64, pages=BUF, most=4, page=16, n_pages=6, stream=0)
    assert set(kw) <= set(a)
    a.update(kw)
    assert _C.lib.lri_attn_prefill_pages(*a.values()) == status
