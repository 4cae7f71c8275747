"""Operators of a paged key-value cache as a serving program calls them, as cases to measure.

store   rows of the fused q/k/v projection: queries and keys rotated by their positions, keys and values written into the pages of their
        sequences, in the activations' type or in 8 bits (e4m3) with a scale for each (position, head)
attend  one new token of each sequence over its pages
load    the pages of some sequences read back into dense caches, which the prompt attention works on

A page holds `page` positions of all key heads.  Sequences own pages in the order that an allocator has left, a table [sequences, most
pages] names them, entries without a page are -1.  Lengths of a batch are spread evenly over the logarithm between the shortest and the
longest; idle rows (a captured step of a larger batch than there are users) have position -1.
"""
import math
import os
import sys

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_E4M3 = torch.float8_e4m3fn
_LARGEST = 448.0       # of e4m3
_SMALLEST = 2.0 ** -100  # a row of smaller values than this is stored against it


# ---- cases --------------------------------------------------------------------------------------------------------------------
def _store(name, dtype, cache, n_head, n_kv, dim, page, seqs, shortest, longest, start, rot, halves, table):
    """`seqs` sequences of shortest..longest new tokens each, behind `start` earlier positions."""
    return {"name": name, "op": "store", "dtype": dtype, "cache": cache, "n_head": n_head, "n_kv": n_kv, "dim": dim, "page": page,
            "seqs": seqs, "shortest": shortest, "longest": longest, "start": start, "rot": rot, "halves": halves, "table": table}


def _attend(name, dtype, cache, n_head, n_kv, dim, page, seqs, shortest, longest, idle=0, window=0):
    return {"name": name, "op": "attend", "dtype": dtype, "cache": cache, "n_head": n_head, "n_kv": n_kv, "dim": dim, "page": page,
            "seqs": seqs, "shortest": shortest, "longest": longest, "idle": idle, "window": window}


def _load(name, dtype, cache, n_kv, dim, page, seqs, shortest, longest):
    return {"name": name, "op": "load", "dtype": dtype, "cache": cache, "n_kv": n_kv, "dim": dim, "page": page, "seqs": seqs,
            "shortest": shortest, "longest": longest}


def listed():
    return [
        # one user of the 8B shape, one new token: nothing but latency
        _store("store-step-1", "bf16", "same", 32, 8, 128, 16, 1, 1, 1, 1024, 128, False, "same"),
        # a served batch with an 8-bit cache, halves of a part of the head rotated, table in 32 bits
        _store("store-step-48-e4m3", "bf16", "e4m3", 32, 8, 128, 32, 48, 1, 1, 700, 64, True, "fp32"),
        # three short prompts of ragged length of the 110M shape, every head with keys of its own, from 8-bit storage
        _store("store-ragged-fp16-e4m3", "fp16", "e4m3", 12, 12, 64, 24, 3, 333, 1001, 0, 64, True, "fp32"),
        # a long prompt of the 8B shape
        _store("store-prompt-8k", "bf16", "same", 32, 8, 128, 64, 1, 8192, 8192, 0, 128, False, "same"),
        # one user of the 8B shape behind a prompt of 1024 tokens: latency
        _attend("attend-1", "bf16", "same", 32, 8, 128, 16, 1, 1025, 1025),
        # a captured step of 24 rows of which five are idle, short and long users side by side
        _attend("attend-24-ragged", "bf16", "same", 32, 8, 128, 32, 24, 17, 8000, idle=5),
        # the type of the reference's driver, every head with keys of its own, a page of an odd size, a sliding window
        _attend("attend-40-fp16-window", "fp16", "same", 24, 24, 128, 24, 40, 200, 3000, window=1000),
        # a large batch with an 8-bit cache
        _attend("attend-100-e4m3", "bf16", "e4m3", 32, 8, 128, 64, 100, 300, 6000),
        # one user with a document of 128 K tokens in an 8-bit cache: the work of one sequence spread over the GPU
        _attend("attend-128k-e4m3", "bf16", "e4m3", 64, 8, 128, 128, 1, 131072, 131072),
        # the 1B shape: heads of 64, a large batch of short users
        _attend("attend-200-narrow", "bf16", "same", 32, 8, 64, 16, 200, 40, 900),
        # the cache of one user in front of the next portion of a prompt
        _load("load-1", "bf16", "same", 8, 128, 16, 1, 1500, 1500),
        # eight users at once, 8 bits back to 16
        _load("load-8-e4m3", "fp16", "e4m3", 8, 128, 64, 8, 500, 16000),
    ]


def draw(rng):
    def spread(lo, hi):
        return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))

    op = rng.choice(("store", "attend", "attend", "load"))
    dtype, cache = rng.choice(("bf16", "fp16")), rng.choice(("same", "e4m3"))
    n_kv, group = rng.choice(((8, 4), (8, 8), (12, 1), (24, 1), (4, 4), (2, 4), (1, 8), (8, 2), (3, 5)))
    dim, page = rng.choice((64, 128, 128, 80)), rng.choice((16, 16, 32, 64, 128, 24, 8))
    if op == "store":
        seqs = spread(1, 64)
        if rng.random() < 0.5:
            shortest = longest = 1
        else:
            longest = spread(2, 8192 // seqs)
            shortest = max(1, longest // rng.choice((1, 2, 7)))
        c = _store("", dtype, cache, n_kv * group, n_kv, dim, page, seqs, shortest, longest, rng.choice((0, spread(1, 4000))),
                   rng.choice((dim, dim, dim // 2)), rng.random() < 0.5, rng.choice(("same", "fp32")))
    elif op == "attend":
        seqs = spread(1, 200)
        longest = spread(1, min(131072, 100_000_000 // (seqs * n_kv * dim)))
        shortest = max(1, longest // rng.choice((1, 2, 30)))
        c = _attend("", dtype, cache, n_kv * group, n_kv, dim, page, seqs, shortest, longest, idle=rng.choice((0, 0, min(seqs - 1, 3))),
                    window=rng.choice((0, 0, 0, spread(1, 4096))))
    else:
        seqs = spread(1, 16)
        longest = spread(1, min(65536, 40_000_000 // (n_kv * dim)) // seqs)
        c = _load("", dtype, cache, n_kv, dim, page, seqs, max(1, longest // rng.choice((1, 3, 20))), longest)
    del c["name"]
    return c


def _lengths(case):
    """New tokens (store) or positions (attend, load) of each sequence; 0 for an idle row."""
    n, lo, hi = case["seqs"], case["shortest"], case["longest"]
    got = [max(lo, min(hi, round(lo * (hi / lo) ** ((i * 0.6180339887498949) % 1)))) for i in range(n)]
    got[0] = hi
    idle = case.get("idle", 0)
    for i in range(idle):
        got[(i + 1) * n // (idle + 1) if idle + 1 < n else n - 1 - i] = 0
    return got


def _visible(case):
    """Positions that the new token of each sequence sees."""
    w = case.get("window", 0)
    return [min(n, w) if w else n for n in _lengths(case)]


def work(case):
    t, c = 2, 1 if case["cache"] == "e4m3" else 2
    n_kv, dim = case["n_kv"], case["dim"]
    row = 2 * n_kv * (dim * c + (4 if c == 1 else 0))  # a position in the cache: keys, values, their scales
    pages = sum(-(-(n + case.get("start", 0)) // case["page"]) for n in _lengths(case)) * 4
    if case["op"] == "store":
        n, nh = sum(_lengths(case)), case["n_head"]
        table = case["longest"] * case["rot"] * (2 if case["table"] == "same" else 4)
        return {"bytes": n * ((2 * nh + 2 * n_kv) * dim * t + row + 8) + table + pages, "flops": n * (nh + n_kv) * case["rot"] * 3}
    if case["op"] == "attend":
        n, nh = sum(_visible(case)), case["n_head"]
        return {"bytes": n * row + case["seqs"] * (2 * nh * dim * t + 4) + pages, "flops": 4 * nh * dim * n}
    n = sum(_lengths(case))
    return {"bytes": n * (row + 2 * n_kv * dim * t) + pages, "flops": 2 * n_kv * dim * n if c == 1 else 0}


# ---- inputs ---------------------------------------------------------------------------------------------------------------------
def _pages(case, lengths, g):
    """The table of pages, in an allocator's order, and how many pages there are."""
    page = case["page"]
    need = [-(-n // page) for n in lengths]
    total, most = sum(need), max(need) + 2
    ids = torch.randperm(total, generator=g).to(torch.int32)
    table = torch.full((len(need), most), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = ids[at:at + n]
        at += n
    return table.cuda(), total


def _cache_values(shape, dtype, seed, spread):
    """What a layer's keys (channels of unequal size) or values (much alike) hold."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(shape, device="cuda", generator=g, dtype=dtype)
    channel = torch.exp(spread * torch.randn((shape[1], 1, shape[3]), device="cuda", generator=g))
    return x.mul_(channel.to(dtype))


def _quantise(x):
    """Codes and scales of rows: the cache that an earlier call has written."""
    top = x.float().abs().amax(-1).clamp_(min=_SMALLEST)
    return (x.float() * (_LARGEST / top).unsqueeze(-1)).clamp_(-_LARGEST, _LARGEST).to(_E4M3), top / _LARGEST


def prepare(case, seed):
    g = torch.Generator().manual_seed(seed)
    gc = torch.Generator(device="cuda").manual_seed(seed)
    dtype, n_kv, dim, page = _TYPES[case["dtype"]], case["n_kv"], case["dim"], case["page"]
    lengths, start = _lengths(case), case.get("start", 0)
    s = {"case": case}
    s["pages"], total = _pages(case, [n + start for n in lengths], g)
    eight = case["cache"] == "e4m3"
    shape = (total, n_kv, page, dim)
    if case["op"] == "store":
        # zeros, so that what the call leaves alone can be told
        k, v = (torch.zeros(shape, dtype=_E4M3 if eight else dtype, device="cuda") for _ in range(2))
        ks, vs = (torch.zeros(shape[:3], device="cuda") if eight else None for _ in range(2))
        heads, n = case["n_head"] + 2 * n_kv, sum(lengths)
        size = torch.exp(0.5 * torch.randn(heads * dim, device="cuda", generator=gc))
        s["qkv"] = (torch.randn(n, heads * dim, device="cuda", generator=gc) * size).to(dtype)
        s["input_pos"] = torch.cat([torch.arange(start, start + m, dtype=torch.int32) for m in lengths]).cuda()
        s["sequence"] = None if case["longest"] == 1 else torch.repeat_interleave(
            torch.arange(len(lengths), dtype=torch.int32), torch.tensor(lengths)).cuda()
        at = torch.arange(start + case["longest"], dtype=torch.float64)
        freq = 500000.0 ** -(torch.arange(0, case["rot"], 2, dtype=torch.float64) / case["rot"])
        angle = torch.outer(at, freq)
        s["table"] = torch.stack([angle.cos(), angle.sin()], -1).to(dtype if case["table"] == "same" else torch.float32).cuda()
    else:
        k, v = _cache_values(shape, dtype, 2 * seed, 0.5), _cache_values(shape, dtype, 2 * seed + 1, 0.1)
        ks = vs = None
        if eight:
            k, ks = _quantise(k)
            v, vs = _quantise(v)
        s["input_pos"] = torch.tensor(lengths, dtype=torch.int32).sub_(1).cuda()
        if case["op"] == "attend":
            s["q"] = torch.randn(case["seqs"], case["n_head"], dim, device="cuda", generator=gc).to(dtype)
        else:
            rows = -(-case["longest"] // 64) * 64
            s["k_out"], s["v_out"] = (torch.zeros(case["seqs"], n_kv, rows, dim, dtype=dtype, device="cuda") for _ in range(2))
    s["k"], s["v"], s["k_scale"], s["v_scale"] = k, v, ks, vs
    if own:  # the cache object and the workspace that a program keeps
        package = os.path.abspath("ladder-residual-inference_b200")
        if package not in sys.path:
            sys.path.insert(0, package)
        from gpt_fast import PagedKVCache
        cache = PagedKVCache(total, page, n_kv, dim, dtype, cache_dtype=_E4M3 if eight else dtype, device="cuda")
        cache.k_pages, cache.v_pages = k, v
        if eight:
            cache.k_scale, cache.v_scale = ks, vs
        s["cache"] = cache
        if case["op"] == "attend":
            s["workspace"] = cache.attend_workspace(case["n_head"])
    return s


# ---- the passes -------------------------------------------------------------------------------------------------------------------
def run(s):
    case = s["case"]
    if own:
        cache = s["cache"]
        if case["op"] == "store":
            q = cache.store(s["qkv"], s["table"], s["input_pos"], s["pages"], case["n_head"], sequence=s["sequence"], halves=case["halves"])
            return {"q": q, "k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
        if case["op"] == "attend":
            return cache.attend(s["q"], s["input_pos"], s["pages"], window=case["window"], workspace=s["workspace"])
        return cache.load(s["input_pos"], s["pages"], out=(s["k_out"], s["v_out"]))
    return {"store": _plain_store, "attend": _plain_attend, "load": _plain_load}[case["op"]](s)


def _rotate(x, c, s, rot, halves):
    """x [tokens, heads, dim] in fp32; c, s [tokens, 1, rot / 2]"""
    if halves:
        x0, x1 = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([x0 * c - x1 * s, x1 * c + x0 * s], -1)
    else:
        x0, x1 = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([x0 * c - x1 * s, x1 * c + x0 * s], -1).flatten(-2)
    return torch.cat([turned, x[..., rot:]], -1)


def _bytes(t):
    return t.view(torch.uint8) if t.dtype == _E4M3 else t


def _plain_store(s):
    case = s["case"]
    nh, n_kv, dim, page = case["n_head"], case["n_kv"], case["dim"], case["page"]
    x = s["qkv"].float().view(-1, nh + 2 * n_kv, dim)
    pos = s["input_pos"].long()
    seq = torch.arange(x.shape[0], device=x.device) if s["sequence"] is None else s["sequence"].long()
    turn = s["table"][pos].float().unsqueeze(1)
    q, k = (_rotate(part, turn[..., 0], turn[..., 1], case["rot"], case["halves"]) for part in (x[:, :nh], x[:, nh:nh + n_kv]))
    v = x[:, nh + n_kv:]
    at = s["pages"][seq, pos // page].long(), pos % page
    for new, pages, scales in ((k, s["k"], s["k_scale"]), (v, s["v"], s["v_scale"])):
        if scales is not None:
            top = new.abs().amax(-1).clamp(min=_SMALLEST)
            scales[at[0], :, at[1]] = top / _LARGEST
            new = (new * (_LARGEST / top).unsqueeze(-1)).clamp(-_LARGEST, _LARGEST)
        _bytes(pages)[at[0], :, at[1]] = _bytes(new.to(pages.dtype))
    return {"q": q.to(s["qkv"].dtype), "k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _gather(s, most):
    """Keys and values of positions 0 .. most - 1 of every sequence in fp32, [sequences, positions, heads, dim]; what has no page may be anything."""
    page = s["case"]["page"]
    at = torch.arange(most, device="cuda")
    ids = s["pages"][:, at // page].long().clamp(min=0)
    for pages, scales in ((s["k"], s["k_scale"]), (s["v"], s["v_scale"])):
        x = _bytes(pages)[ids, :, at % page]
        yield x.float() if scales is None else x.view(_E4M3).float() * scales[ids, :, at % page].unsqueeze(-1)


def _plain_attend(s):
    case = s["case"]
    q, n_kv, most = s["q"].float(), case["n_kv"], case["longest"]
    k, v = _gather(s, most)
    q = q.view(q.shape[0], n_kv, -1, q.shape[-1])
    scores = torch.einsum("bhgd,bjhd->bhgj", q, k) * case["dim"] ** -0.5
    at, pos = torch.arange(most, device="cuda"), s["input_pos"].long().view(-1, 1)
    seen = at <= pos
    if case["window"]:
        seen &= at > pos - case["window"]
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    weights = (scores - scores.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)).exp()
    total = weights.sum(-1, keepdim=True)
    y = torch.einsum("bhgj,bjhd->bhgd", weights, v) / torch.where(total > 0, total, 1.0)
    return y.reshape(s["q"].shape).to(s["q"].dtype)


def _plain_load(s):
    at = torch.arange(s["case"]["longest"], device="cuda")
    there = (at <= s["input_pos"].long().view(-1, 1))[..., None, None]
    for x, out in zip(_gather(s, s["case"]["longest"]), (s["k_out"], s["v_out"])):
        out[:, :, :at.numel()] = torch.where(there, x, 0.0).to(out.dtype).transpose(1, 2)
    return s["k_out"], s["v_out"]


# ---- from the definition, in 64 bits ------------------------------------------------------------------------------------------------
def _nearest_e4m3(y):
    """y, |y| <= 448, at the nearest number of three mantissa bits, ties to even; steps of 2^-9 below 2^-6."""
    _, e = torch.frexp(y.abs())
    step = torch.ldexp(torch.ones_like(y), (e - 1).clamp(min=-6) - 3)
    return torch.round(y / step) * step


def _exact_store(s):
    case = s["case"]
    nh, n_kv, dim, page, rot = (case[k] for k in ("n_head", "n_kv", "dim", "page", "rot"))
    x = s["qkv"].double().unflatten(1, (nh + 2 * n_kv, dim))
    turn = s["table"].double()[s["input_pos"].long()]
    z = torch.complex(turn[..., 0], turn[..., 1]).unsqueeze(1)
    qk = x[:, :nh + n_kv]
    pair = qk[..., :rot].unflatten(-1, (2, rot // 2)).transpose(-1, -2) if case["halves"] else qk[..., :rot].unflatten(-1, (rot // 2, 2))
    turned = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * z)
    turned = (turned.transpose(-1, -2) if case["halves"] else turned).flatten(-2)
    qk = torch.cat([turned, qk[..., rot:]], -1)
    got = {"q": qk[:, :nh], "k_scale": None, "v_scale": None}
    seq = s["sequence"] if s["sequence"] is not None else torch.arange(x.shape[0], device="cuda")
    page_of = s["pages"].long()[seq.long(), torch.div(s["input_pos"], page, rounding_mode="floor").long()]
    row = page_of * page + s["input_pos"].long() % page
    for name, new in (("k", qk[:, nh:]), ("v", x[:, nh + n_kv:])):
        whole = torch.zeros(s[name].shape[0] * page, n_kv, dim, dtype=torch.float64, device="cuda")
        if s["k_scale"] is not None:
            top = new.abs().amax(-1, keepdim=True).clamp(min=_SMALLEST)
            scales = torch.zeros(whole.shape[:2], dtype=torch.float64, device="cuda")
            scales[row] = top[..., 0] / _LARGEST
            got[name + "_scale"] = scales.view(-1, page, n_kv).transpose(1, 2)
            new = _nearest_e4m3(new / top * _LARGEST)
        whole[row] = new
        got[name] = whole.view(-1, page, n_kv, dim).transpose(1, 2)
    return got


def _exact_rows(s, b, lo, hi):
    """Keys and values of positions lo .. hi - 1 of sequence b, [heads, positions, dim]."""
    page = s["case"]["page"]
    at = torch.arange(lo, hi, device="cuda")
    ids = s["pages"][b].long()[torch.div(at, page, rounding_mode="floor")]
    for name in ("k", "v"):
        x = _bytes(s[name])[ids, :, at % page].view(s[name].dtype).double()
        if s[name + "_scale"] is not None:
            x *= s[name + "_scale"][ids, :, at % page].double().unsqueeze(-1)
        yield x.transpose(0, 1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "store":
        return _exact_store(s)
    if case["op"] == "attend":
        y = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        for b, (n, seen) in enumerate(zip(_lengths(case), _visible(case))):
            if n:
                k, v = _exact_rows(s, b, n - seen, n)
                q = s["q"][b].double().unflatten(0, (case["n_kv"], -1))
                y[b] = (torch.softmax(q @ k.transpose(1, 2) / math.sqrt(case["dim"]), -1) @ v).flatten(0, 1)
        return y
    outs = [torch.zeros(s["k_out"].shape, dtype=torch.float64, device="cuda") for _ in range(2)]
    for b, n in enumerate(_lengths(case)):
        for out, x in zip(outs, _exact_rows(s, b, 0, n)):
            out[b, :, :n] = x
    return tuple(outs)
