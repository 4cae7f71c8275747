"""Prompt attention over a copy of a sequence's pages, where positions and pages are missing, against its definition in 64 bits."""
import pytest
import torch

from paged_util import TINY, half_step, make_cache

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _no_wait_gave_up():
    yield
    from gpt_fast import _C
    torch.cuda.synchronize()
    _C.check(_C.lib.lri_gemm_status())


@pytest.fixture(params=[1, 0], ids=["tcgen05", "mma"])
def kernel(request):
    from gpt_fast import _C
    _C.check(_C.lib.lri_set_option(b"attn_prefill_tc", request.param))
    yield
    _C.check(_C.lib.lri_set_option(b"attn_prefill_tc", 1))


def _prompt_64(q, k, v, pos, named):
    """q [tokens, heads, dim] over rows k, v [KV heads, rows, dim] of which `named` have pages: the result in 64 bits and how far a right one may be off.
    Probabilities and the result are rounded to the type once (half a step of what they weigh), scores are sums in 32 bits (dim + 2 roundings of the sum of
    magnitudes), 2^-18 is for the exponentials and the sums over positions.  Halves end at steps of 2^-24: a probability, the largest at least 1, is off by up
    to 2^-25 however small it is."""
    group, dim, half = q.shape[1] // k.shape[0], q.shape[2], half_step(q.dtype)
    seen = (torch.arange(k.shape[1], device="cuda") <= pos.long()[:, None]) & named
    qd, kd, vd = q.double().transpose(0, 1), *(torch.where(named[:, None], t.double(), 0.0).repeat_interleave(group, 0) for t in (k, v))
    w = torch.softmax((qd @ kd.transpose(1, 2) * dim ** -0.5).masked_fill(~seen, -torch.inf), -1).nan_to_num(0.0)
    loose = (qd.abs() @ kd.abs().transpose(1, 2) * dim ** -0.5).amax() * (dim + 2) * 2.0 ** -24
    y = w @ vd
    tol = (w @ vd.abs()) * (half + 2 * loose + 2.0 ** -18) + half * y.abs() + TINY[q.dtype]
    if q.dtype == torch.float16:
        tol += 2.0 ** -25 * (seen.double() @ vd.abs())
    return y.transpose(0, 1), tol.transpose(0, 1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("n_head,n_kv,dim", [(8, 2, 64), (4, 4, 128)])
@pytest.mark.parametrize("page,length,start,S,gone", [
    (16, 70, 0, 70, []), (8, 300, 100, 200, [0, 1, 2, 20, 21]), (64, 200, 0, 200, [0]), (24, 130, 127, 3, [0, 1, 2, 3, 4]), (16, 500, 360, 140, [22, 23, 24, 30]),
    (128, 1000, 488, 512, [0, 1, 3]), (40, 64, 0, 64, [0, 1]), (16, 33, 31, 2, [])])
def test_pages_that_are_missing(dtype, eight, n_head, n_kv, dim, page, length, start, S, gone, kernel):
    from gpt_fast.ops import CudaOps
    cache, table = make_cache([length], page, n_kv, dim, dtype, eight, seed=length)
    for i, p in enumerate(gone):
        table[0, p] = -1 if i % 2 else cache.k_pages.shape[0]
    rows = -(-length // 64) * 64 + 64
    k, v = (torch.full((1, n_kv, rows, dim), float("nan"), dtype=dtype, device="cuda") for _ in range(2))  # what was left by others
    pos = torch.arange(start, start + S, device="cuda")
    cache.load(pos[-1:], table, out=(k, v))
    q = torch.randn(S, n_head, dim, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).to(dtype)
    named = (table[0] >= 0) & (table[0] < cache.k_pages.shape[0])
    named = torch.nn.functional.pad(named.repeat_interleave(page), (0, rows))[:rows]
    want, tol = _prompt_64(q, k[0], v[0], pos, named)
    for at in (pos, pos.int()):
        out = torch.full((S, n_head * dim), float("nan"), dtype=dtype, device="cuda")
        CudaOps.attention_pages(q, k, v, at, table, page, cache.k_pages.shape[0], out, S, n_head, n_kv, dim)
        assert ((out.view(S, n_head, dim).double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dim", [64, 128])
def test_positions_of_any_order(dim, kernel):
    """Tokens without a position among the others, whole tiles of them, positions behind the pages (the last counts), the same position twice; the largest
    and the smallest of 64 bits."""
    from gpt_fast.ops import CudaOps
    dtype, page, n_head, n_kv, length, S = torch.bfloat16, 16, 6, 3, 290, 400
    cache, table = make_cache([length], page, n_kv, dim, dtype, False)
    table = table[:, :18].contiguous()  # 288 positions
    k, v = (torch.full((1, n_kv, 320, dim), float("nan"), dtype=dtype, device="cuda") for _ in range(2))
    pos = torch.full((S,), -1, dtype=torch.int64)
    pos[:100] = torch.randperm(288, generator=torch.Generator().manual_seed(0))[:100]
    pos[7], pos[8], pos[9], pos[10], pos[11] = -1, 2 ** 63 - 1, -2 ** 63, 288, pos[12]
    pos[380:] = torch.arange(20)
    pos = pos.cuda()
    cache.load(pos.amax(0, keepdim=True), table, out=(k, v))
    q = torch.randn(S, n_head, dim, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).to(dtype)
    named = torch.arange(320, device="cuda") < 288
    want, tol = _prompt_64(q, k[0], v[0], pos, named)
    out = torch.full((S, n_head * dim), float("nan"), dtype=dtype, device="cuda")
    CudaOps.attention_pages(q, k, v, pos, table, page, cache.k_pages.shape[0], out, S, n_head, n_kv, dim)
    got = out.view(S, n_head, dim)
    assert ((got.double() - want).abs() <= tol).all() and not got[100:380].any() and not got[[7, 9]].any()


@pytest.mark.parametrize("S", [2, 70, 128, 300])
def test_whole_prompts_as_the_dense_kernel(S, kernel):
    """With every page there and positions that follow one another: the same bits as dense prompt attention."""
    from gpt_fast.ops import CudaOps
    dtype, page, n_head, n_kv, dim = torch.bfloat16, 32, 4, 2, 128
    cache, table = make_cache([S + 33], page, n_kv, dim, dtype, False)
    pos = torch.arange(33, S + 33, device="cuda")
    k, v = (torch.zeros(1, n_kv, 384, dim, dtype=dtype, device="cuda") for _ in range(2))
    cache.load(pos[-1:], table, out=(k, v))
    q = torch.randn(S, n_head, dim, device="cuda").to(dtype)
    a, b = (torch.empty(S, n_head * dim, dtype=dtype, device="cuda") for _ in range(2))
    CudaOps.attention_pages(q, k, v, pos, table, page, cache.k_pages.shape[0], a, S, n_head, n_kv, dim)
    CudaOps.attention(q, k, v, pos, b, 1, S, n_head, n_kv, dim, None, 1)
    assert torch.equal(a, b)
