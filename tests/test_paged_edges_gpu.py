"""The paged operators at the ends of what they take."""
import pytest
import torch

from paged_util import E4M3, attend_64, make_cache

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _no_wait_gave_up():
    yield
    from gpt_fast import _C
    torch.cuda.synchronize()
    _C.check(_C.lib.lri_gemm_status())


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("n_head,n_kv,dim,window", [(8, 8, 128, 0), (40, 2, 128, 0), (32, 32, 64, 0), (8, 8, 128, 4096)])
def test_attend_tables_of_2_to_the_30_positions(eight, n_head, n_kv, dim, window):
    """The widest tables that are allowed, and short sequences in them."""
    lengths, page = [5000, 0, 100], 4096
    cache, table = make_cache(lengths, page, n_kv, dim, torch.bfloat16, eight)
    wide = torch.full((3, 2 ** 30 // page), -1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    q = torch.randn(3, n_head, dim, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(torch.bfloat16)
    pos = torch.tensor(lengths, dtype=torch.int32, device="cuda") - 1
    want, tol = attend_64(cache, table, q, lengths, window)
    assert ((cache.attend(q, pos, wide, window=window).double() - want).abs() <= tol).all()


@pytest.mark.parametrize("eight", [False, True])
def test_a_single_row_has_no_pitch(eight):
    """One token, one sequence: the strides of their rows may be any numbers."""
    from gpt_fast import PagedKVCache
    n_head, n_kv, dim, page, dtype = 4, 2, 64, 16, torch.bfloat16
    width = (n_head + 2 * n_kv) * dim
    x = torch.randn(2, width + 4, device="cuda").to(dtype)
    table = torch.tensor([2, 0, 1], dtype=torch.int32, device="cuda")
    pos = torch.tensor([17], dtype=torch.int32, device="cuda")
    got = []
    for qkv, pages in ((x[:1, :width].clone(), table[None]), (x[:1, :width], table[None]), (x[0, :width].clone()[:, None].t(), table[:, None].t()),
                       (x[0, :width].as_strided((1, width), (0, 1)), table.as_strided((1, 3), (1, 1)))):
        cache = PagedKVCache(3, page, n_kv, dim, dtype, cache_dtype=E4M3 if eight else dtype, device="cuda")
        q = cache.store(qkv, None, pos, pages, n_head)
        got.append((q, cache.k_pages.view(torch.uint8), cache.attend(q, pos, pages)) + cache.load(pos, pages))
    for other in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(other, got[0]))
