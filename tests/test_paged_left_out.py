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
