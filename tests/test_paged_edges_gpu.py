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
