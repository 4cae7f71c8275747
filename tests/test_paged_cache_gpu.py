"""The operators of the paged key-value cache against their definitions in 64 bits."""
import math

import pytest
import torch

from paged_util import E4M3, TINY, attend_64, dense, half_step, make_cache, rotate_64, table_for

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16]


@pytest.fixture(autouse=True)
def _no_wait_gave_up():
    yield
    from gpt_fast import _C
    torch.cuda.synchronize()
    _C.check(_C.lib.lri_gemm_status())


# ---- store -----------------------------------------------------------------------------------------------------------------------
def _store_case(dtype, eight, n_head, n_kv, dim, page, starts, counts, rot, halves, table_type, seed=0):
    from gpt_fast import PagedKVCache
    g = torch.Generator(device="cuda").manual_seed(seed)
    tokens = sum(counts)
    qkv = (torch.randn(tokens, (n_head + 2 * n_kv) * dim, device="cuda", generator=g) * 3).to(dtype)
    pos = torch.cat([torch.arange(s, s + n, dtype=torch.int32) for s, n in zip(starts, counts)]).cuda()
    seq = torch.repeat_interleave(torch.arange(len(counts), dtype=torch.int32), torch.tensor(counts)).cuda()
    pages, n_pages = table_for([s + n for s, n in zip(starts, counts)], page, seed=seed)
    rope = None
    if rot:
        angle = torch.outer(torch.arange(max(s + n for s, n in zip(starts, counts))).double(), 10000.0 ** -(torch.arange(rot // 2).double() * 2 / rot))
        rope = torch.stack([angle.cos(), angle.sin()], -1).to(table_type).cuda()
    cache = PagedKVCache(n_pages, page, n_kv, dim, dtype, cache_dtype=E4M3 if eight else dtype, device="cuda")
    return cache, qkv, rope, pos, pages, seq


def _check_store(cache, q, qkv, rope, pos, pages, seq, n_head, halves, live=None):
    n_kv, page, dim = cache.k_pages.shape[1:]
    dtype, tokens = qkv.dtype, qkv.shape[0]
    live = torch.ones(tokens, dtype=torch.bool, device="cuda") if live is None else live
    x = qkv.double().view(tokens, n_head + 2 * n_kv, dim)[live]
    rot = 0 if rope is None else 2 * rope.shape[1]
    qk, size = x[:, :n_head + n_kv], x[:, :n_head + n_kv].abs()
    if rot:
        qk, size = rotate_64(qk, rope[pos.long()[live]], rot, halves)
    loose = size * 2.0 ** -22  # products and their sum in 32 bits
    want_q = qk[:, :n_head]
    assert ((q[live].double() - want_q).abs() <= want_q.abs() * half_step(dtype) + loose[:, :n_head] + TINY[dtype]).all()
    p, s = pos.long()[live], seq.long()[live]
    ids, rows = pages[s, p // page].long(), p % page
    for name, want, off in (("k", qk[:, n_head:], loose[:, n_head:]), ("v", x[:, n_head + n_kv:], torch.zeros_like(x[:, n_head + n_kv:]))):
        stored, scales = getattr(cache, name + "_pages"), getattr(cache, name + "_scale")
        got = stored.view(torch.uint8 if scales is not None else dtype)[ids, :, rows].view(stored.dtype).double()
        if scales is None:
            assert ((got - want).abs() <= want.abs() * half_step(dtype) + off + TINY[dtype]).all()
            if name == "v":
                assert torch.equal(got, want)
            continue
        scale = scales[ids, :, rows].double()[..., None]
        top = want.abs().amax(-1, keepdim=True)
        assert ((scale - top / 448).abs() <= top / 448 * 2.0 ** -23 + off.amax(-1, keepdim=True) / 448 + 2.0 ** -108).all()
        # half a step of e4m3: 2^-4 of the value, of the smallest numbers 2^-10 of the scale
        assert ((got * scale - want).abs() <= want.abs() * (2.0 ** -4 + 2.0 ** -20) + scale * 2.0 ** -10 + off).all()
    # nothing else was written
    touched = torch.zeros(cache.k_pages.shape[0], page, dtype=torch.bool, device="cuda")
    touched[ids, rows] = True
    for t in (cache.k_pages, cache.v_pages):
        assert not t.view(torch.uint8).view(t.shape[0], n_kv, page, -1).transpose(1, 2)[~touched].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("n_head,n_kv,dim,page,rot,halves,table_type", [
    (32, 8, 128, 16, 128, False, None), (32, 8, 128, 32, 128, True, torch.float32), (12, 12, 64, 24, 32, True, None), (4, 2, 80, 8, 20, False, torch.float32),
    (6, 1, 48, 16, 36, True, None), (3, 3, 256, 64, 64, False, torch.float32), (5, 1, 8, 8, 0, False, None), (2, 2, 104, 128, 2, True, torch.float32)])
@pytest.mark.parametrize("counts,starts", [([1], [0]), ([1, 1, 1, 1, 1], [0, 7, 8, 1000, 31]), ([37, 1, 130], [0, 5, 100])])
def test_store(dtype, eight, n_head, n_kv, dim, page, rot, halves, table_type, counts, starts):
    cache, qkv, rope, pos, pages, seq = _store_case(dtype, eight, n_head, n_kv, dim, page, starts, counts, rot, halves, table_type or dtype)
    one_each = all(n == 1 for n in counts)
    q = cache.store(qkv, rope, pos, pages, n_head, sequence=None if one_each else seq, halves=halves)
    _check_store(cache, q, qkv, rope, pos, pages, seq, n_head, halves)


@pytest.mark.parametrize("eight", [False, True])
def test_store_skips_tokens_without_a_place(eight):
    """Negative positions, positions behind the table or the pages, sequences and pages that do not exist: not written, the query row neither;
    positions in 64 bits, a strided row, a table with a pitch."""
    dtype, n_head, n_kv, dim, page = torch.bfloat16, 4, 2, 64, 16
    cache, qkv, rope, pos, pages, seq = _store_case(dtype, eight, n_head, n_kv, dim, page, [0, 3], [40, 20], 64, False, dtype)
    wide = torch.zeros(pages.shape[0], pages.shape[1] + 3, dtype=torch.int32, device="cuda")
    wide[:, :pages.shape[1]] = pages
    pages = wide[:, :pages.shape[1]]
    pages[0, 1] = -1
    pages[1, 1] = cache.k_pages.shape[0]
    pos = pos.long()
    pos[2], pos[3], pos[4], pos[5] = -1, 10 ** 12, rope.shape[0], pages.shape[1] * page
    seq[6], seq[7] = -1, 2
    live = torch.ones(60, dtype=torch.bool, device="cuda")
    live[[2, 3, 4, 5, 6, 7]] = False
    live &= torch.tensor([not (s == 0 and p // 16 == 1) and not (s == 1 and p // 16 == 1) for s, p in zip(seq.tolist(), pos.tolist())], device="cuda")
    padded = torch.zeros(60, qkv.shape[1] + 8, dtype=dtype, device="cuda")
    padded[:, :qkv.shape[1]] = qkv
    out = torch.full((60, n_head, dim), 7.0, dtype=dtype, device="cuda")
    cache.store(padded[:, :qkv.shape[1]], rope, pos, pages, n_head, sequence=seq, out=out)
    assert (out[~live] == 7).all()
    _check_store(cache, out, qkv, rope, pos, pages, seq, n_head, False, live)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("rot", [0, 8])
def test_store_many_tokens_of_few_heads(eight, rot):
    """Blocks with more tokens than threads."""
    dtype, n_head, n_kv, dim = torch.bfloat16, 1, 1, 8
    cache, qkv, rope, pos, pages, seq = _store_case(dtype, eight, n_head, n_kv, dim, 64, [0, 9, 100], [30000, 1, 5003], rot, False, dtype)
    pos[17::1000] = -1
    live = pos >= 0
    q = cache.store(qkv, rope, pos, pages, n_head, sequence=seq)
    _check_store(cache, q, qkv, rope, pos, pages, seq, n_head, False, live)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("tokens", [5, 700])
def test_store_behind_a_kernel_that_writes_what_it_reads(eight, tokens):
    """Positions, sequence numbers, pages and angles come from the kernels directly in front, which let this one begin before they are done: two sets in
    turn, copied as the bits of a small cache's rows (a `load`), never waited for on the host."""
    from gpt_fast import PagedKVCache
    n_head, n_kv, dim, page, most, dtype = 4, 2, 64, 16, 16, torch.bfloat16
    notes = PagedKVCache(2, 64, 1, 64, dtype, device="cuda")  # keys: the pages' table, then positions and sequences as bits; values: unused
    angles = PagedKVCache(2, 256, 1, 64, dtype, device="cuda")
    g = torch.Generator().manual_seed(0)
    per = -(-tokens // 4)
    sets = []
    for i in range(2):
        pages = torch.randperm(4 * most, generator=g).to(torch.int32).view(4, most)
        pages[i, 3] = -1
        at = torch.arange(4 * per)
        seq, pos = ((at // per + i) % 4).to(torch.int32)[:tokens], (at % per + 5 + 20 * i).to(torch.int32)[:tokens]
        pos[1 + i] = -1
        words = torch.zeros(64 * 32, dtype=torch.int32)
        words[:64], words[64:64 + tokens], words[1024:1024 + tokens] = pages.view(-1), pos, seq
        notes.k_pages[i, 0] = words.view(dtype).view(64, 64).cuda()
        angles.k_pages[i, 0] = torch.randn(256, 64, generator=g).to(dtype).cuda()
        sets.append((pages.cuda(), pos.cuda(), seq.cuda(), angles.k_pages[i, 0].view(256, 32, 2)))
    which = [torch.tensor([[i]], dtype=torch.int32, device="cuda") for i in range(2)]
    last = torch.tensor([255], dtype=torch.int32, device="cuda")
    words, spare = (torch.zeros(1, 1, 64, 64, dtype=dtype, device="cuda") for _ in range(2))
    rope, spare2 = (torch.zeros(1, 1, 256, 64, dtype=dtype, device="cuda") for _ in range(2))
    w = words.view(torch.int32).view(-1)
    qkv = (torch.randn(tokens, (n_head + 2 * n_kv) * dim, generator=g) * 3).to(dtype).cuda()
    caches = [PagedKVCache(4 * most, page, n_kv, dim, dtype, cache_dtype=E4M3 if eight else dtype, device="cuda") for _ in range(12)]
    got = []
    torch.cuda.synchronize()
    for n, cache in enumerate(caches):
        loads = [lambda i=n % 2: notes.load(last, which[i], out=(words, spare)), lambda i=n % 2: angles.load(last, which[i], out=(rope, spare2))]
        for load in loads if n % 4 < 2 else loads[::-1]:
            load()
        got.append(cache.store(qkv, rope.view(256, 32, 2), w[64:64 + tokens], w[:64].view(4, most), n_head, sequence=w[1024:1024 + tokens]))
    for n, (cache, q) in enumerate(zip(caches, got)):
        pages, pos, seq, table = sets[n % 2]
        live = (pos >= 0) & (pages[seq.long(), pos.clamp(min=0).long() // page] >= 0)
        _check_store(cache, q, qkv, table, pos, pages, seq, n_head, False, live)


def test_store_values_at_the_edges_of_e4m3():
    """Rows of zeros, of the smallest and largest numbers, with an infinity or a NaN."""
    from gpt_fast import PagedKVCache
    dtype, dim = torch.bfloat16, 64
    rows = torch.zeros(6, dim)
    rows[1] = 2.0 ** -133
    rows[2] = 3.38e38
    rows[3] = torch.linspace(-1, 1, dim)
    rows[3, 5] = float("inf")
    rows[4] = 1.0
    rows[4, 63] = float("nan")
    rows[5, 0], rows[5, 1], rows[5, 2] = 448.0, 2.0 ** -9, 1.5 * 2.0 ** -9  # scale 1: the smallest code, and a tie above it (to even: 2)
    qkv = torch.cat([rows, rows, rows], 1).to(dtype).cuda()
    cache = PagedKVCache(1, 8, 1, dim, dtype, cache_dtype=E4M3, device="cuda")
    pages = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    cache.store(qkv, None, torch.arange(6, dtype=torch.int32, device="cuda"), pages, 1, sequence=torch.zeros(6, dtype=torch.int32, device="cuda"))
    for name in ("k", "v"):
        codes, scale = getattr(cache, name + "_pages")[0, 0].float().cpu(), getattr(cache, name + "_scale")[0, 0].cpu()
        assert not codes[0].any() and scale[0] > 0 and not codes[1].any()
        assert (codes[2] == 448).all() and scale[2].isfinite()
        assert scale[3].isnan() and scale[4].isnan()
        assert scale[5] == 1 and codes[5, :3].tolist() == [448.0, 2.0 ** -9, 2 * 2.0 ** -9]
        assert not codes[6:].any() and not scale[6:].any()


# ---- attend ----------------------------------------------------------------------------------------------------------------------
def _attend(cache, table, q, lengths, **kw):
    pos = torch.tensor(lengths, dtype=torch.int32, device="cuda") - 1
    out = torch.full_like(q, float("nan"))
    return cache.attend(q, pos, table, out=out, **kw)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("n_head,n_kv,dim", [(32, 8, 128), (12, 12, 64), (8, 1, 64), (20, 1, 128), (10, 2, 80), (3, 3, 72), (34, 2, 48), (16, 1, 128), (4, 2, 192),
                                             (2, 2, 8), (6, 2, 16), (3, 1, 24), (9, 1, 112)])
@pytest.mark.parametrize("page,lengths,window", [
    (16, [1], 0), (8, [0, 1, 7, 8, 9, 31, 32, 33], 0), (24, [500, 0, 23, 24, 25, 129, 1], 0), (64, [1025, 3], 0), (128, [2000, 1, 65, 0], 100),
    (8, [257, 64, 40], 1), (40, [300, 41, 1000], 64), (16, [5000], 0), (4096, [4097, 4096, 1], 0)])
def test_attend(dtype, eight, n_head, n_kv, dim, page, lengths, window):
    cache, table = make_cache(lengths, page, n_kv, dim, dtype, eight, seed=n_head + page)
    q = torch.randn(len(lengths), n_head, dim, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5)).to(dtype)
    want, tol = attend_64(cache, table, q, lengths, window)
    ws = cache.attend_workspace(n_head)
    got = _attend(cache, table, q, lengths, window=window, workspace=ws)
    assert ((got.double() - want).abs() <= tol).all()
    assert torch.equal(got, _attend(cache, table, q, lengths, window=window, workspace=ws))  # left ready, and the same bits again


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("seqs", [1, 3, 40, 200])
def test_attend_many_lengths(eight, seqs):
    """Batches whose sequences end anywhere in the runs of the GPU's CTAs."""
    g = torch.Generator().manual_seed(seqs)
    for n_head, n_kv, dim, most in ((32, 8, 128, 3000 // seqs + 100), (4, 4, 64, 40000 // seqs)):
        lengths = torch.randint(0, most, (seqs,), generator=g).tolist()
        cache, table = make_cache(lengths, 16, n_kv, dim, torch.bfloat16, eight, seed=seqs)
        q = torch.randn(seqs, n_head, dim, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(torch.bfloat16)
        want, tol = attend_64(cache, table, q, lengths)
        assert ((_attend(cache, table, q, lengths, workspace=cache.attend_workspace(n_head)).double() - want).abs() <= tol).all()


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("dim", [64, 128, 192])
def test_attend_pages(eight, dim):
    """Pages that are missing or do not exist are left out; sequences share pages; a table with a pitch; a position behind the table's pages counts
    as its last; positions in 64 bits; a scale of one's own."""
    lengths = [100, 300, 64, 200]
    cache, table = make_cache(lengths, 16, 2, dim, torch.bfloat16, eight)
    wide = torch.full((4, table.shape[1] + 5), 2 ** 31 - 1, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    table = wide[:, :table.shape[1]]
    table[0, 2] = -1
    table[1, 0] = cache.k_pages.shape[0]
    table[1, 5] = -2 ** 31
    table[2, :] = -1
    table[3, :4] = table[1, 1:5]
    q = torch.randn(4, 8, dim, device="cuda").to(torch.bfloat16)
    pos = torch.tensor([99, 299, 63, 199], dtype=torch.int64, device="cuda")
    want, tol = attend_64(cache, table, q, lengths, scale=0.3)
    got = cache.attend(q, pos, table, scale=0.3)
    assert ((got.double() - want).abs() <= tol).all() and not got[2].any()
    full = [table.shape[1] * 16, 0, 0, 0]
    cache2, table2 = make_cache(full, 16, 2, dim, torch.bfloat16, eight)
    table2 = table2[:, :table.shape[1]].contiguous()
    want, tol = attend_64(cache2, table2, q, full)
    got = cache2.attend(q, torch.tensor([10 ** 12, -5, -10 ** 12, -1], dtype=torch.int64, device="cuda"), table2)
    assert ((got.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("dim", [128, 192])
def test_attend_values_that_are_not_finite(eight, dim):
    """A NaN in a visible row reaches the sequence's results and no other's; scores of 1e4 and equal scores."""
    lengths = [50, 70, 33, 64]
    cache, table = make_cache(lengths, 16, 1, dim, torch.bfloat16, eight)
    q = torch.randn(4, 4, dim, device="cuda").to(torch.bfloat16)
    q[2] = 0
    q[3] *= 1000
    page = table[1, 2].item()
    (cache.v_scale if eight else cache.v_pages)[page, 0, 3] = float("nan")
    got = _attend(cache, table, q, lengths)
    assert got[1].isnan().all()
    keep = [0, 2, 3]
    want, tol = attend_64(cache, table, q, lengths)
    assert ((got.double() - want).abs() <= tol)[keep].all()


def test_attend_captured_and_advanced_in_place():
    """A captured store and attention replayed while positions grow, and a page is added, in place."""
    dtype, n_head, n_kv, dim, page = torch.bfloat16, 8, 2, 128, 16
    lengths = [30, 5, 0]
    cache, table = make_cache([64, 64, 64], page, n_kv, dim, dtype, True)
    table[0, 2:] = -1
    pos = torch.tensor(lengths, dtype=torch.int32, device="cuda") - 1
    ws = cache.attend_workspace(n_head)
    qkv = torch.randn(3, (n_head + 2 * n_kv) * dim, device="cuda").to(dtype)
    out = torch.zeros(3, n_head, dim, dtype=dtype, device="cuda")
    q = torch.zeros_like(out)

    def step():
        pos.add_((pos >= 0).int())
        cache.store(qkv, None, pos, table, n_head, out=q)
        cache.attend(q, pos, table, out=out, workspace=ws)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    owned = table.clone()
    spare = [i for i in range(cache.k_pages.shape[0]) if i not in owned.flatten().tolist()]
    for n in range(4):
        if n == 1:
            table[0, 2] = spare[0]
        qkv.copy_(torch.randn_like(qkv.float()).to(dtype))
        graph.replay()
        now = [31 + n + 1, 6 + n + 1, 0]
        assert pos.tolist() == [x - 1 for x in now]
        want, tol = attend_64(cache, table, q, now)
        assert ((out.double() - want).abs() <= tol).all()


def test_attend_two_graphs_share_a_workspace():
    """Captured calls of unequal batches that share a workspace, replayed in turn."""
    ws, graphs = None, []
    for lengths, n_head in (([3000, 17, 900], 8), ([40] * 50, 16), ([9000], 8)):
        cache, table = make_cache(lengths, 32, 2, 128, torch.bfloat16, False, seed=len(lengths))
        q = torch.randn(len(lengths), n_head, 128, device="cuda").to(torch.bfloat16)
        pos = torch.tensor(lengths, dtype=torch.int32, device="cuda") - 1
        ws = cache.attend_workspace(16) if ws is None else ws
        out = torch.zeros_like(q)
        cache.attend(q, pos, table, out=out, workspace=ws)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            cache.attend(q, pos, table, out=out, workspace=ws)
        graphs.append((graph, out) + attend_64(cache, table, q, lengths) + (cache, table, q, pos))
    for _ in range(3):
        for graph, out, want, tol, *_ in graphs:
            out.zero_()
            graph.replay()
            assert ((out.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("dim", [128, 192])
def test_attend_behind_a_kernel_that_writes_its_table(eight, dim):
    """Table and positions come from the kernel directly in front, which lets this one begin before it is done: two tables in turn, copied as the
    bits of a small cache's rows (a `load`), never waited for on the host."""
    from gpt_fast import PagedKVCache
    lengths = [[700, 40, 1300, 0], [32, 1200, 64, 333]]
    cache, table = make_cache([max(a, b) for a, b in zip(*lengths)], 16, 2, dim, torch.bfloat16, eight)
    order = [table, table[:, [1, 0] + list(range(2, table.shape[1]))].contiguous()]  # the second's first two pages change places
    most = 128  # entries of a sequence: four rows of 32 numbers
    notes = PagedKVCache(2, 16, 1, 64, torch.bfloat16, device="cuda")  # a page's rows hold a table as bits, its values' first row the positions
    for i in range(2):
        wide = torch.full((4, most), -1, dtype=torch.int32, device="cuda")
        wide[:, :table.shape[1]] = order[i]
        notes.k_pages[i, 0] = wide.view(torch.bfloat16).view(16, 64)
        at = torch.full((32,), -1, dtype=torch.int32, device="cuda")
        at[:4] = torch.tensor(lengths[i], dtype=torch.int32, device="cuda") - 1
        notes.v_pages[i, 0, 0] = at.view(torch.bfloat16)
    which = [torch.tensor([[i]], dtype=torch.int32, device="cuda") for i in range(2)]
    last = torch.tensor([15], dtype=torch.int32, device="cuda")
    out = tuple(torch.zeros(1, 1, 16, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    pages, pos = out[0].view(torch.int32).view(4, most), out[1].view(torch.int32).view(-1)[:4]
    q = torch.randn(4, 8, dim, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).to(torch.bfloat16)
    ws = cache.attend_workspace(8)
    want = [attend_64(cache, order[i], q, lengths[i]) for i in range(2)]
    got = []
    for n in range(30):
        notes.load(last, which[n % 2], out=out)
        got.append(cache.attend(q, pos, pages, workspace=ws))
    for n, y in enumerate(got):
        assert ((y.double() - want[n % 2][0]).abs() <= want[n % 2][1]).all()


def test_attend_on_another_stream():
    lengths = [700, 20, 1300]
    cache, table = make_cache(lengths, 16, 4, 128, torch.bfloat16, True)
    q = torch.randn(3, 8, 128, device="cuda").to(torch.bfloat16)
    want, tol = attend_64(cache, table, q, lengths)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = _attend(cache, table, q, lengths)
    torch.cuda.current_stream().wait_stream(stream)
    assert ((got.double() - want).abs() <= tol).all()


def test_attend_on_two_streams_at_once():
    """Calls that may overlap on the device, each with a workspace of its own: the same bits as one behind the other."""
    cases = []
    for seed, lengths in ((1, [3000, 40, 900]), (2, [17, 2500])):
        cache, table = make_cache(lengths, 16, 8, 128, torch.bfloat16, False, seed=seed)
        q = torch.randn(len(lengths), 32, 128, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(torch.bfloat16)
        pos = torch.tensor([n - 1 for n in lengths], dtype=torch.int32, device="cuda")
        cases.append((cache, q, pos, table, cache.attend_workspace(32), torch.cuda.Stream()))
    want = [cache.attend(q, pos, table, workspace=ws) for cache, q, pos, table, ws, _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, (cache, q, pos, table, ws, stream) in enumerate(cases):
            with torch.cuda.stream(stream):
                got[i].append(cache.attend(q, pos, table, workspace=ws))
    torch.cuda.synchronize()
    for y, w in zip(got, want):
        assert all(torch.equal(x, w) for x in y)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("dim", [128, 192])
@pytest.mark.parametrize("scale", [0.0, -0.2])
def test_attend_scales_that_are_not_positive(eight, dim, scale):
    lengths = [300, 1, 40]
    cache, table = make_cache(lengths, 16, 2, dim, torch.bfloat16, eight)
    q = torch.randn(3, 8, dim, device="cuda", generator=torch.Generator(device="cuda").manual_seed(4)).to(torch.bfloat16)
    want, tol = attend_64(cache, table, q, lengths, scale=scale)
    got = cache.attend(q, torch.tensor([n - 1 for n in lengths], dtype=torch.int32, device="cuda"), table, scale=scale)
    assert ((got.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dim", [128, 192])
def test_positions_at_the_ends_of_64_bits(dim):
    """The largest position is one behind the pages (attention and reading back: all of them; storing: left out), the smallest an idle row."""
    cache, table = make_cache([48, 48], 16, 2, dim, torch.bfloat16, False)
    table = table[:, :3]
    pos = torch.tensor([2 ** 63 - 1, -2 ** 63], dtype=torch.int64, device="cuda")
    q = torch.randn(2, 4, dim, device="cuda", generator=torch.Generator(device="cuda").manual_seed(6)).to(torch.bfloat16)
    want, tol = attend_64(cache, table, q, [48, 0])
    got = cache.attend(q, pos, table)
    assert ((got.double() - want).abs() <= tol).all() and not got[1].any()
    k, v = cache.load(pos, table)
    for x, y in zip((k, v), dense(cache, table, 0, 0, 48)):
        assert torch.equal(x[0].double(), y) and not x[1].any()
    before, out = cache.k_pages.clone(), torch.full((2, 4, dim), 7.0, dtype=torch.bfloat16, device="cuda")
    cache.store(torch.randn(2, 8 * dim, device="cuda").to(torch.bfloat16), None, pos, table, 4, out=out)
    assert torch.equal(before.view(torch.int16), cache.k_pages.view(torch.int16)) and (out == 7).all()


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("dim", [64, 192])
def test_attend_more_sequences_than_a_launch_takes(eight, dim):
    lengths = [(7 * i) % 40 for i in range(1100)]
    cache, table = make_cache(lengths, 8, 1, dim, torch.bfloat16, eight)
    q = torch.randn(1100, 2, dim, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).to(torch.bfloat16)
    want, tol = attend_64(cache, table, q, lengths)
    assert ((_attend(cache, table, q, lengths).double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dim", [128, 160])
def test_offsets_beyond_32_bits(dim):
    """A cache of more than 2^31 elements, the sequence's pages at its end: stored, read by attention, read back."""
    n_kv, page, n_head, n = 8, 64, 16, 150
    n_pages = 2 ** 31 // (n_kv * page * dim) + 64
    from gpt_fast import PagedKVCache
    cache = PagedKVCache(n_pages, page, n_kv, dim, torch.bfloat16, cache_dtype=E4M3, device="cuda")
    table = torch.tensor([[n_pages - 1, n_pages - 9, n_pages - 4]], dtype=torch.int32, device="cuda")
    qkv = torch.randn(n, (n_head + 2 * n_kv) * dim, device="cuda", generator=torch.Generator(device="cuda").manual_seed(0)).to(torch.bfloat16)
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    q = cache.store(qkv, None, pos, table, n_head, sequence=torch.zeros(n, dtype=torch.int32, device="cuda"))
    k, v = dense(cache, table, 0, 0, n)
    x = qkv.double().view(n, n_head + 2 * n_kv, dim).transpose(0, 1)
    for got, want in ((k, x[n_head:n_head + n_kv]), (v, x[n_head + n_kv:])):
        # half a step of e4m3: 2^-4 of the value, of the smallest numbers 2^-10 of the scale
        assert ((got - want).abs() <= want.abs() * (2.0 ** -4 + 2.0 ** -20) + want.abs().amax(-1, keepdim=True) / 448 * 2.0 ** -10 * (1 + 2.0 ** -20)).all()
    last = q[n - 1:].contiguous()
    want, tol = attend_64(cache, table, last, [n])
    assert ((cache.attend(last, pos[n - 1:], table).double() - want).abs() <= tol).all()
    back = cache.load(pos[n - 1:], table)
    assert ((back[0][0, :, :n].double() - k).abs() <= k.abs() * half_step(torch.bfloat16) * (1 + 2.0 ** -8)).all()
    assert ((back[1][0, :, :n].double() - v).abs() <= v.abs() * half_step(torch.bfloat16) * (1 + 2.0 ** -8)).all()
    # and nothing in front of them
    assert not any(int(t.view(torch.uint8)[: n_pages - 9].amax()) for t in (cache.k_pages, cache.v_pages))


# ---- load ------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("n_kv,dim,page", [(8, 128, 16), (3, 64, 24), (1, 80, 8), (2, 256, 128), (2, 8, 8)])
@pytest.mark.parametrize("lengths", [[1], [0, 63, 64, 65], [500, 1, 129]])
def test_load(dtype, eight, n_kv, dim, page, lengths):
    cache, table = make_cache(lengths, page, n_kv, dim, dtype, eight)
    table[0, 0] = -1  # a page that is missing reads as zeros
    rows = 70 if max(lengths) > 70 else max(lengths) + 200
    out = tuple(torch.full((len(lengths), n_kv, rows, dim), 7.0, dtype=dtype, device="cuda") for _ in range(2))
    last = torch.tensor(lengths, dtype=torch.int64, device="cuda") - 1
    assert cache.load(last, table, out=out) is out
    for b, n in enumerate(lengths):
        n = min(n, rows)
        gap = min(n, page) if b == 0 else 0
        for got, want in zip(out, dense(cache, table, b, gap, n)):
            assert not got[b, :, :gap].any()
            if eight:
                assert ((got[b, :, gap:n].double() - want).abs() <= want.abs() * (half_step(dtype) + 2.0 ** -24) * (1 + 2.0 ** -10) + TINY[dtype]).all()
            else:
                assert torch.equal(got[b, :, gap:n].double(), want)
            assert not got[b, :, n:-(-n // 64) * 64].any()
            assert (got[b, :, -(-n // 64) * 64:] == 7).all()


def test_load_makes_its_caches():
    lengths = [20, 0, 33]
    cache, table = make_cache(lengths, 16, 2, 64, torch.float16, False)
    last = torch.tensor(lengths, dtype=torch.int32, device="cuda") - 1
    k, v = cache.load(last, table)
    assert k.shape == (3, 2, table.shape[1] * 16, 64) and not k[1].any() and not v[2, :, 33:].any()
    k2, v2 = cache.load(last, table, rows=24)
    assert torch.equal(k2, k[:, :, :24]) and torch.equal(v2, v[:, :, :24])


# ---- a run of them -----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("eight", [False, True])
def test_prompt_then_steps(dtype, eight):
    """Ragged prompts stored together, read back for the dense prompt attention, then steps of all sequences, against dense attention over what
    the cache holds and over the values themselves."""
    from gpt_fast.ops import CudaOps as ops
    n_head, n_kv, dim, page, counts = 8, 2, 64, 16, [130, 1, 57]
    cache, qkv, rope, pos, _, seq = _store_case(dtype, eight, n_head, n_kv, dim, page, [0, 0, 0], counts, dim, False, dtype)
    pages, n_pages = table_for([n + 40 for n in counts], page)
    from gpt_fast import PagedKVCache
    cache = PagedKVCache(n_pages, page, n_kv, dim, dtype, cache_dtype=E4M3 if eight else dtype, device="cuda")
    q = cache.store(qkv, rope, pos, pages, n_head, sequence=seq)
    last = torch.tensor(counts, dtype=torch.int32, device="cuda") - 1
    k, v = cache.load(last, pages)
    at = 0
    for b, n in enumerate(counts):
        out = torch.empty(n, n_head * dim, dtype=dtype, device="cuda")
        qb = q[at:at + n].contiguous()
        if n > 1:
            ops.attention(qb, k[b:b + 1], v[b:b + 1], torch.arange(n, dtype=torch.int32, device="cuda"), out, 1, n, n_head, n_kv, dim, None, 1)
            kk, vv = (t[b, :, :n].double().repeat_interleave(n_head // n_kv, 0) for t in (k, v))
            s = qb.double().transpose(0, 1) @ kk.transpose(1, 2) * dim ** -0.5
            w = torch.softmax(s.masked_fill(torch.ones(n, n, device="cuda").triu(1).bool(), -math.inf), -1)
            want, size = (w @ vv).transpose(0, 1), (w @ vv.abs()).transpose(0, 1)
            # probabilities, and the sum that divides, in the type; values read back and the result rounded once
            assert ((out.view(n, n_head, dim).double() - want).abs() <= size * 4 * half_step(dtype)).all()
        at += n
    lengths = list(counts)
    table = torch.stack([torch.cos(torch.outer(torch.arange(200.0), 10000.0 ** -(torch.arange(0, dim, 2) / dim))),
                         torch.sin(torch.outer(torch.arange(200.0), 10000.0 ** -(torch.arange(0, dim, 2) / dim)))], -1).to(dtype).cuda()
    ws = cache.attend_workspace(n_head)
    for step in range(5):
        rows = torch.randn(3, (n_head + 2 * n_kv) * dim, device="cuda", generator=torch.Generator(device="cuda").manual_seed(step)).to(dtype)
        now = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        lengths = [n + 1 for n in lengths]
        q = cache.store(rows, table, now, pages, n_head)
        want, tol = attend_64(cache, pages, q, lengths)
        assert ((cache.attend(q, now, pages, workspace=ws).double() - want).abs() <= tol).all()
