"""The paged operators at the ends of what they take."""
import pytest
import torch

from paged_util import E4M3, TINY, attend_64, half_step, make_cache

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


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("dim,rot,tokens", [(64, 64, 3), (128, 0, 700), (80, 20, 64), (192, 64, 65)])
def test_fresh_queries_hold_nothing_of_other_memory(eight, dim, rot, tokens):
    """Without `out`, the rows of tokens that are left out are zeros, whatever lay in the memory before; an `out` of the caller's keeps them."""
    from gpt_fast import PagedKVCache
    n_head, n_kv, page, dtype = 3, 1, 16, torch.bfloat16
    x = torch.randn(tokens, (n_head + 2 * n_kv) * dim, device="cuda").to(dtype)
    rope = torch.randn(tokens, rot // 2, 2, device="cuda").to(dtype) if rot else None
    per = -(-tokens // page)
    table = torch.arange(per, dtype=torch.int32, device="cuda")[None].clone()
    table[0, -1] = -1
    pos, seq = torch.arange(tokens, dtype=torch.int32, device="cuda"), torch.zeros(tokens, dtype=torch.int32, device="cuda")
    pos[::5] = -1
    live = (pos >= 0) & (table[0, pos.clamp(min=0).long() // page] >= 0)
    cache = PagedKVCache(per, page, n_kv, dim, dtype, cache_dtype=E4M3 if eight else dtype, device="cuda")
    kept = torch.full((tokens, n_head, dim), 7.0, dtype=dtype, device="cuda")
    cache.store(x, rope, pos, table, n_head, sequence=seq, out=kept)
    for _ in range(3):
        torch.full((tokens, n_head, dim), float("nan"), dtype=dtype, device="cuda")  # freed at once: the next allocation finds it
        q = cache.store(x, rope, pos, table, n_head, sequence=seq)
        assert not q[~live].any() and torch.equal(q[live], kept[live])
    assert (kept[~live] == 7).all()


# ---- what the other tests would not notice -------------------------------------------------------------------------------------------
def _cancelling(dtype, eight, dim, n, seqs, group):
    """Sequences of n positions whose values cancel: the result is far smaller than what it is made of, so that the rounding of probabilities shows.  The
    last position weighs most and has minus the sum of the others over its own weight.  Queries and keys are multiples of 1/8 up to 2, whose products and
    sums 32 bits hold exactly; e4m3: codes of values are 1, the values their scales."""
    g = torch.Generator(device="cuda").manual_seed(n)
    q = (torch.randint(-8, 9, (seqs, 1, dim), device="cuda", generator=g) / 4).to(dtype)
    k = torch.randint(-8, 9, (seqs, n, dim), device="cuda", generator=g) / 4
    k[:, -1] = q[:, 0].float() / 2
    s = (q.double() @ k.double().transpose(1, 2)).squeeze(1) * dim ** -0.5
    w = torch.softmax(s, -1)
    kind = torch.float32 if eight else dtype  # of values
    v = (torch.rand(seqs, n, 1 if eight else dim, device="cuda", generator=g) + 0.5).to(kind).double()
    v[:, -1] = -(w[:, :-1, None] * v[:, :-1]).sum(1).div(w[:, -1:]).to(kind).double()
    page = 16
    per = -(-n // page)
    from gpt_fast import PagedKVCache
    cache = PagedKVCache(seqs * per, page, 1, dim, dtype, cache_dtype=E4M3 if eight else dtype, device="cuda")
    table = torch.randperm(seqs * per, device="cuda").to(torch.int32).view(seqs, per)
    at = torch.arange(n, device="cuda")
    ids = table.long()[:, at // page]
    if eight:
        cache.k_pages.view(torch.uint8)[ids, 0, at % page] = k.to(E4M3).view(torch.uint8)
        cache.v_pages.view(torch.uint8).fill_(0x38)
        cache.k_scale.fill_(1)
        cache.v_scale[ids, 0, at % page] = v[..., 0].float()
    else:
        cache.k_pages[ids, 0, at % page], cache.v_pages[ids, 0, at % page] = k.to(dtype), v.to(dtype)
    return cache, table, q.expand(seqs, group, dim).contiguous(), s, w, v.expand(seqs, n, dim)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("dim,n,group", [(128, 3, 4), (64, 24, 8), (128, 40, 16), (64, 40, 3)])
def test_probabilities_keep_their_digits(dtype, eight, dim, n, group):
    """Probabilities enter the second product as the sum of two 16-bit numbers, off by half a step of half a step (bf16 2^-16, halves 2^-22) of what they
    are; rounded once they would be off by more than is allowed here, which is checked too.

    Scores are exact up to their scale (four roundings of 2^-24, of a probability and of the sum that divides), exponentials are off by 2^-22 (twice for the same
    reason, and once for a reference that moved), sums over the positions by a rounding each, e4m3 by six for the values' scales, the result by its own
    rounding.  Halves end at steps of 2^-24: 2^-34 of the largest value a position."""
    cache, table, q, s, w, v = _cancelling(dtype, eight, dim, n, 48, group)
    kind = torch.float16 if eight else dtype
    want, size = (w[:, None] @ v)[:, 0], (w[:, None] @ v.abs())[:, 0]
    off = half_step(kind) ** 2 + 2 * 4 * s.abs().amax().item() * 2.0 ** -24 + 3 * 2.0 ** -22 + (n + 8) * 2.0 ** -24 + 6 * 2.0 ** -24
    tol = size * off + half_step(dtype) * want.abs() + TINY[dtype]
    if kind == torch.float16:
        tol = tol + n * 2.0 ** -34 * v.abs().amax(1)
    got = cache.attend(q, torch.full((48,), n - 1, dtype=torch.int32, device="cuda"), table)
    assert ((got.double() - want[:, None]).abs() <= tol[:, None]).all()
    p = (s - s.amax(-1, keepdim=True)).exp()
    if eight:
        top = v[..., 0].abs().amax(-1, keepdim=True)
        once = ((p * v[..., 0] / top * 2.0 ** 9).to(kind).double() * top * 2.0 ** -9).sum(-1, keepdim=True)
    else:
        once = ((p * 2.0 ** 9).to(kind).double()[:, None] @ v)[:, 0] * 2.0 ** -9
    assert ((once / p.sum(-1, keepdim=True) - want).abs() > tol).any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_codes_are_the_nearest(dtype):
    """e4m3 codes of values (which do not rotate) by whole numbers: 448 |x| and code * top are exact in 64 bits, and no other code is nearer; ties go to
    the even one."""
    from gpt_fast import PagedKVCache
    n, dim, page = 500, 128, 32
    x = (torch.randn(n, 3 * dim, device="cuda", generator=torch.Generator(device="cuda").manual_seed(0)) * 3).to(dtype)
    x[:, 2 * dim] = x[:, 2 * dim:].abs().amax(-1)
    x[::4, 2 * dim] = 7.0  # largest magnitudes whose quotients hit midpoints
    x[::4, 2 * dim + 1:] = x[::4, 2 * dim + 1:].clamp(-6.5, 6.5)
    cache = PagedKVCache(16, page, 1, dim, dtype, cache_dtype=E4M3, device="cuda")
    table = torch.arange(16, dtype=torch.int32, device="cuda")[None]
    cache.store(x, None, torch.arange(n, dtype=torch.int32, device="cuda"), table, 1, sequence=torch.zeros(n, dtype=torch.int32, device="cuda"))
    v = x[:, 2 * dim:].double()
    top = v.abs().amax(-1, keepdim=True)
    codes = cache.v_pages.view(torch.uint8)[:, 0].reshape(-1, dim)[:n].long()
    size, sign = codes & 127, codes >> 7
    assert ((sign == 1) == (v < 0))[size > 0].all() and size.amax() == 126
    numbers = torch.arange(128, dtype=torch.uint8, device="cuda").view(E4M3).double()
    numbers[127] = torch.inf
    far = lambda c: (448 * v.abs() - numbers[c] * top).abs()  # noqa: E731
    off, below, above = far(size), far((size - 1).clamp(min=0)), far(size + 1)
    below[size == 0] = torch.inf
    assert (off <= below).all() and (off <= above).all()
    ties = (off == below) | (off == above)
    assert ties.any() and (size[ties] % 2 == 0).all()


@pytest.mark.parametrize("eight", [False, True])
def test_store_writes_nothing_else(eight):
    """Codes and scales of all other rows, and query rows of tokens without a place, stay as they were."""
    from gpt_fast import PagedKVCache
    n_head, n_kv, dim, page, dtype = 4, 3, 80, 24, torch.float16
    cache = PagedKVCache(9, page, n_kv, dim, dtype, cache_dtype=E4M3 if eight else dtype, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(0)
    for t in cache.buffers():
        t.view(torch.uint8).copy_(torch.randint(0, 256, t.view(torch.uint8).shape, device="cuda", generator=g).to(torch.uint8))
    before = [t.view(torch.uint8).clone() for t in cache.buffers()]
    counts, pos = [30, 1, 51], torch.cat([torch.arange(s, s + n) for s, n in ((0, 30), (71, 1), (3, 51))]).int().cuda()
    seq = torch.repeat_interleave(torch.arange(3, dtype=torch.int32), torch.tensor(counts)).cuda()
    table = torch.tensor([[8, 1, -1], [2, 3, 4], [5, 9, 7]], dtype=torch.int32, device="cuda")
    pos[4], pos[40] = -1, 72
    ids = table[seq.long(), (pos.long() // page).clamp(0, 2)].long()
    live = (pos >= 0) & (pos < 72) & (ids >= 0) & (ids < 9)
    x = torch.randn(82, (n_head + 2 * n_kv) * dim, device="cuda", generator=g).to(dtype)
    out = torch.full((82, n_head, dim), 7.0, dtype=dtype, device="cuda")
    cache.store(x, None, pos, table, n_head, sequence=seq, out=out)
    touched = torch.zeros(9, page, dtype=torch.bool, device="cuda")
    touched[ids[live], pos.long()[live] % page] = True
    assert 0 < touched.sum() == live.sum() and (out[~live] == 7).all() and torch.equal(out[live], x.view(82, -1, dim)[live, :n_head])
    for t, b in zip(cache.buffers(), before):
        now = t.view(torch.uint8).view(9, n_kv, page, -1).transpose(1, 2)
        assert torch.equal(now[~touched], b.view(9, n_kv, page, -1).transpose(1, 2)[~touched])


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("dim", [8, 136, 192])
def test_attend_more_sequences_than_a_grid_has(dim, eight):
    """65535 in a launch of the plain kernel, 1024 in one of the other: sequences of up to eight positions that share a page."""
    n, dtype = 2 * 65535 + 11, torch.bfloat16
    cache, _ = make_cache([8], 8, 1, dim, dtype, eight)
    page = int((~(cache.k_scale if eight else cache.k_pages[..., 0])[:, 0].isnan().any(-1)).nonzero()[0])
    table = torch.full((n, 1), page, dtype=torch.int32, device="cuda")
    pos = (torch.arange(n, device="cuda") % 9).int() - 1
    q = torch.randn(n, 2, dim, device="cuda", generator=torch.Generator(device="cuda").manual_seed(0)).to(dtype)
    got = cache.attend(q, pos, table)
    for p in range(-1, 8):
        rows = pos == p
        few = q[rows]
        want, tol = attend_64(cache, table[:1], few.transpose(0, 1).reshape(1, -1, dim), [p + 1])  # all as heads of one sequence
        want, tol = (t.view(2, -1, dim).transpose(0, 1) for t in (want, tol))
        assert ((got[rows].double() - want).abs() <= tol).all()
