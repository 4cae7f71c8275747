"""Paged caches for tests: random contents with everything that no sequence owns poisoned, and the operators' definitions in 64 bits."""
import torch

E4M3 = torch.float8_e4m3fn
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}  # half a step of the smallest numbers


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def table_for(lengths, page, spare=1, seed=0, device="cuda", pitch=0):
    """Pages of sequences of these lengths in a random order, -1 behind them; the number of pages (three belong to nobody)."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lengths]
    ids = torch.randperm(sum(need) + 3, generator=g).to(torch.int32)
    most = max(need) + spare
    table = torch.full((len(need), most + pitch), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = ids[at:at + n]
        at += n
    return table.to(device)[:, :most], sum(need) + 3


def make_cache(lengths, page, n_kv, dim, dtype, eight, seed=0, device="cuda"):
    """A PagedKVCache whose rows behind the sequences' ends and whose free pages hold NaN; the table; dense (k, v) lists in 64 bits."""
    from gpt_fast import PagedKVCache
    table, n_pages = table_for(lengths, page, seed=seed, device=device)
    cache = PagedKVCache(n_pages, page, n_kv, dim, dtype, cache_dtype=E4M3 if eight else dtype, device=device)
    g = torch.Generator(device=device).manual_seed(seed)
    owned = torch.zeros(n_pages, page, dtype=torch.bool, device=device)
    for b, n in enumerate(lengths):
        at = torch.arange(n, device=device)
        owned[table[b, at // page].long(), at % page] = True
    mask = owned[:, None].expand(n_pages, n_kv, page)
    for pages, scales in ((cache.k_pages, cache.k_scale), (cache.v_pages, cache.v_scale)):
        x = torch.randn(pages.shape, device=device, generator=g)
        if eight:
            x = (x * 100).clamp(-448, 448).to(E4M3)
            x.view(torch.uint8)[~mask] = 0x7F
            s = torch.exp(2 * torch.randn(scales.shape, device=device, generator=g)) / 200
            s[~mask] = float("nan")
            scales.copy_(s)
            pages.view(torch.uint8).copy_(x.view(torch.uint8))
        else:
            x[~mask] = float("nan")
            pages.copy_(x.to(dtype))
    return cache, table


def dense(cache, table, b, lo, hi, with_scales=False):
    """Keys and values of positions lo .. hi - 1 of sequence b in 64 bits, [heads, positions, dim]; only positions that have a page."""
    page, n_pages = cache.k_pages.shape[2], cache.k_pages.shape[0]
    at = torch.arange(lo, hi, device=table.device)
    ids = table[b].long()[at // page]
    there = (ids >= 0) & (ids < n_pages)
    at, ids = at[there], ids[there]
    got = []
    for pages, scales in ((cache.k_pages, cache.k_scale), (cache.v_pages, cache.v_scale)):
        x = pages.view(torch.uint8 if scales is not None else pages.dtype)[ids, :, at % page].view(pages.dtype).double()
        s = torch.ones_like(x[..., 0]) if scales is None else scales[ids, :, at % page].double()
        got.append((x * s[..., None]).transpose(0, 1))
    return got + [x.transpose(0, 1), s.transpose(0, 1)] if with_scales else got


def attend_64(cache, table, q, lengths, window=0, scale=None):
    """The result in 64 bits and how far a right one may be off: probabilities rounded once to the type (half a step of what they weigh), sums
    in 32 bits of the scores (dim + 2 roundings of the sum of magnitudes), 2^-18 for the exponentials and the sums over positions, and the
    result's own rounding.

    Probabilities that are halves (fp16 and e4m3 pages) end at steps of 2^-24: taken 2^9 times as large, p (with e4m3 p scale / largest scale) is off by
    up to 2^-25 2^-9 = 2^-34 however small it is.  The largest p is at least 1 in these units, so the sum that divides is too, and the result is off by up
    to 2^-34 times the sum of |value| (e4m3: |code| times the largest scale) over the positions: it shows where all that has weight is zero."""
    n_kv, dim = cache.k_pages.shape[1], cache.k_pages.shape[3]
    scale = dim ** -0.5 if scale is None else scale
    y, tol = torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64)
    half = half_step(q.dtype)
    for b, n in enumerate(lengths):
        n = max(0, min(n, table.shape[1] * cache.k_pages.shape[2]))
        k, v, codes, scales = dense(cache, table, b, max(0, n - window) if window else 0, n, True)
        if k.shape[1] == 0:
            continue
        qb = q[b].double().view(n_kv, -1, dim)
        w = torch.softmax(qb @ k.transpose(1, 2) * scale, -1)
        loose = (qb.abs() @ k.abs().transpose(1, 2) * abs(scale)).amax() * (dim + 2) * 2.0 ** -24
        y[b] = (w @ v).reshape(q[b].shape)
        tol[b] = (w @ v.abs()).reshape(q[b].shape) * (half + 2 * loose + 2.0 ** -18) + half * y[b].abs() + TINY[q.dtype]
        if cache.v_scale is not None or q.dtype == torch.float16:
            ends = 2.0 ** -34 * codes.abs().sum(1) * scales.amax(-1, keepdim=True)
            tol[b] += ends[:, None].expand(-1, qb.shape[1], -1).reshape(q[b].shape)
    return y, tol


def rotate_64(x, angles, rot, halves):
    """x [tokens, heads, dim] in 64 bits, angles [tokens, rot / 2, 2]: the rotated rows, and the magnitudes that their sums are made of."""
    y, size = x.clone(), x.abs().clone()
    c, s = angles[..., 0][:, None].double(), angles[..., 1][:, None].double()
    a, b = (slice(0, rot // 2), slice(rot // 2, rot)) if halves else (slice(0, rot, 2), slice(1, rot, 2))
    x0, x1 = x[..., a], x[..., b]
    y[..., a], y[..., b] = x0 * c - x1 * s, x1 * c + x0 * s
    size[..., a] = size[..., b] = (x0 * c).abs() + (x1 * s).abs() + (x1 * c).abs() + (x0 * s).abs()
    return y, size
