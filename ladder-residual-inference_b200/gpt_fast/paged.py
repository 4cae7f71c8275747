"""Paged key-value cache: keys and values of sequences of unequal lengths that come and go.

A page holds `page_size` positions of all heads; a table [sequences, most pages] (int32, kept by the caller) names the pages of each
sequence in order, with -1 where there is none.  Pages hold the activations' type, or 8 bits (e4m3) with an fp32 scale for each (position, head).
No counterpart in the reference, whose caches are dense and whose batches share their positions (gpt_fast/utils.py:43-59).

Positions, tables and sequence numbers are read on the device: a captured step stays valid when the caller changes them in place.
"""
from typing import Optional, Tuple

import torch
import torch.nn as nn
from torch import Tensor

from .utils import _ops

_INTEGERS = (torch.int32, torch.int64)


def _require(ok, message):
    if not ok:
        raise ValueError(message)


class PagedKVCache(nn.Module):
    """k_pages, v_pages [n_pages, n_heads, page_size, head_dim] in `cache_dtype` (default: dtype), and k_scale, v_scale
    [n_pages, n_heads, page_size] where that is torch.float8_e4m3fn, None otherwise."""

    def __init__(self, n_pages: int, page_size: int, n_heads: int, head_dim: int, dtype: torch.dtype = torch.bfloat16,
                 cache_dtype: Optional[torch.dtype] = None, device=None):
        super().__init__()
        cache_dtype = dtype if cache_dtype is None else cache_dtype
        if dtype not in (torch.bfloat16, torch.float16):
            raise TypeError(f"a paged cache works with bfloat16 or float16 activations, not {dtype}")
        if cache_dtype not in (dtype, torch.float8_e4m3fn):
            raise TypeError(f"pages hold the activations' type ({dtype}) or float8_e4m3fn, not {cache_dtype}")
        _require(n_pages >= 1 and n_heads >= 1, f"{n_pages} pages of {n_heads} heads")
        _require(page_size % 8 == 0 and 8 <= page_size <= 4096, f"page_size={page_size}: a multiple of 8 up to 4096")
        _require(head_dim % 8 == 0 and 8 <= head_dim <= 256, f"head_dim={head_dim}: a multiple of 8 up to 256")
        self.dtype = dtype
        shape = (n_pages, n_heads, page_size, head_dim)
        self.register_buffer("k_pages", torch.zeros(shape, dtype=cache_dtype, device=device))
        self.register_buffer("v_pages", torch.zeros(shape, dtype=cache_dtype, device=device))
        eight = cache_dtype == torch.float8_e4m3fn
        self.register_buffer("k_scale", torch.zeros(shape[:3], device=device) if eight else None)
        self.register_buffer("v_scale", torch.zeros(shape[:3], device=device) if eight else None)

    def _tensors(self):
        b = self._buffers
        k, v, ks, vs = b["k_pages"], b["v_pages"], b["k_scale"], b["v_scale"]
        # (a module cast to another type after its caches were made would hold codes without their meaning)
        _require(k.dtype == v.dtype and k.shape == v.shape and k.is_contiguous() and v.is_contiguous(), "k_pages and v_pages are contiguous and alike")
        if k.dtype == torch.float8_e4m3fn:
            _require(ks is not None and vs is not None and ks.dtype == vs.dtype == torch.float32 and ks.shape == vs.shape == k.shape[:3] and
                     ks.is_contiguous() and vs.is_contiguous(), "e4m3 pages have contiguous fp32 scales [n_pages, n_heads, page_size]")
        else:
            _require(ks is None and vs is None and k.dtype == self.dtype, f"pages hold {self.dtype}, or e4m3 with scales")
        return k, v, ks, vs

    @staticmethod
    def _check(rows, input_pos, pages):
        _require(input_pos.dtype in _INTEGERS and input_pos.shape == (rows,) and input_pos.is_contiguous(),
                 f"positions: {rows} contiguous int32 or int64 numbers, not {input_pos.dtype} {tuple(input_pos.shape)}")
        _require(pages.dtype == torch.int32 and pages.dim() == 2 and pages.shape[1] >= 1 and (pages.stride(1) == 1 or pages.shape[1] == 1),
                 "pages: an int32 table [sequences, most pages] with contiguous rows")

    def store(self, qkv: Tensor, table: Optional[Tensor], input_pos: Tensor, pages: Tensor, n_head: int,
              sequence: Optional[Tensor] = None, halves: bool = False, out: Optional[Tensor] = None) -> Tensor:
        """qkv [tokens, (n_head + 2 n_heads) head_dim], rows [q | k | v heads] of the fused projection: rotates queries and keys by their
        positions, writes keys and values into the pages, returns the queries [tokens, n_head, head_dim].  Token i has position
        input_pos[i] in sequence sequence[i] (None: in sequence i).  table [positions, rot / 2, 2] (cos, sin) in the activations' type or
        fp32, None for no rotation: the first rot elements of a head turn, in adjacent pairs (utils.precompute_freqs_cis) or in halves.
        A token without a position (negative, behind the table) or without a page is left out, its query row too.  One call
        may name a (sequence, position) once."""
        k, v, ks, vs = self._tensors()
        n_kv, dim = k.shape[1], k.shape[3]
        _require(n_head >= 1 and qkv.dim() == 2 and qkv.shape[1] == (n_head + 2 * n_kv) * dim and qkv.dtype == self.dtype and
                 (qkv.stride(1) == 1 or qkv.shape[0] == 0),
                 f"qkv: rows of {n_head} + 2 * {n_kv} heads of {dim} in {self.dtype}, not {qkv.dtype} {tuple(qkv.shape)}")
        tokens = qkv.shape[0]
        self._check(tokens, input_pos, pages)
        _require(tokens == pages.shape[0] if sequence is None else
                 sequence.dtype == torch.int32 and sequence.shape == (tokens,) and sequence.is_contiguous(),
                 f"sequence: {tokens} contiguous int32 numbers, or None for one token of each sequence")
        if table is not None:
            _require(table.dim() == 3 and table.shape[2] == 2 and 2 <= 2 * table.shape[1] <= dim and table.is_contiguous() and
                     table.dtype in (self.dtype, torch.float32), f"table: [positions, rot / 2, 2] in {self.dtype} or float32, rot up to {dim}")
        if out is None:
            out = torch.empty(tokens, n_head, dim, dtype=self.dtype, device=qkv.device)
        else:
            _require(out.dtype == self.dtype and out.shape == (tokens, n_head, dim) and out.is_contiguous(), f"out: [{tokens}, {n_head}, {dim}]")
        _ops().rope_paged_store(qkv, table, input_pos, sequence, pages, out, k, v, ks, vs, n_head, halves)
        return out

    def attend_workspace(self, n_head: int) -> Tensor:
        """The workspace of `attend`: kept by the caller and shared by calls that do not overlap on the device."""
        k = self.k_pages
        return torch.zeros(_ops().paged_attn_workspace_bytes(n_head, k.shape[1], k.shape[3]), dtype=torch.uint8, device=k.device)

    def attend(self, q: Tensor, input_pos: Tensor, pages: Tensor, window: int = 0, scale: Optional[float] = None,
               out: Optional[Tensor] = None, workspace: Optional[Tensor] = None) -> Tensor:
        """Attention of one new token of each sequence, whose row is in the cache: q [sequences, n_head, head_dim] over positions
        0 .. input_pos[b] (the last `window` of them if it is not 0); zeros where that is none.  scale: 1 / sqrt(head_dim) by default.
        workspace: from attend_workspace(n_head); allocated for the call if None."""
        k, v, ks, vs = self._tensors()
        n_kv, dim = k.shape[1], k.shape[3]
        _require(q.dim() == 3 and q.shape[2] == dim and q.shape[1] >= 1 and q.shape[1] % n_kv == 0 and q.dtype == self.dtype and
                 q.is_contiguous(), f"q: contiguous [sequences, a multiple of {n_kv}, {dim}] in {self.dtype}, not {q.dtype} {tuple(q.shape)}")
        self._check(q.shape[0], input_pos, pages)
        _require(pages.shape[0] == q.shape[0], f"pages of {pages.shape[0]} sequences for {q.shape[0]}")
        _require(window >= 0, f"window={window}")
        if workspace is None:
            workspace = self.attend_workspace(q.shape[1])
        if out is None:
            out = torch.empty_like(q)
        else:
            _require(out.dtype == q.dtype and out.shape == q.shape and out.is_contiguous(), f"out: {tuple(q.shape)}")
        _ops().paged_attention(q, k, v, ks, vs, pages, input_pos, window, dim ** -0.5 if scale is None else scale, out, q.shape[1], workspace)
        return out

    def load(self, last_pos: Tensor, pages: Tensor, rows: Optional[int] = None, out: Optional[Tuple[Tensor, Tensor]] = None):
        """Positions 0 .. last_pos[b] of every sequence as dense caches (k, v) [sequences, n_heads, rows, head_dim] in the activations'
        type, as KVCache holds them: what prompt attention works on.  `out` is written in place: rows behind the last position up to
        a multiple of 64 become zeros, later ones stay as they were.  Without it caches of `rows` positions (default: all that the
        table's pages hold) are made, zero behind the last position."""
        k, v, ks, vs = self._tensors()
        n_kv, dim = k.shape[1], k.shape[3]
        self._check(pages.shape[0], last_pos, pages)
        if out is None:
            shape = (pages.shape[0], n_kv, pages.shape[1] * k.shape[2] if rows is None else rows, dim)
            out = torch.zeros(shape, dtype=self.dtype, device=k.device), torch.zeros(shape, dtype=self.dtype, device=k.device)
        k_out, v_out = out
        for t in out:
            _require(t.dtype == self.dtype and t.dim() == 4 and t.shape == k_out.shape and t.is_contiguous() and
                     t.shape[0] == pages.shape[0] and t.shape[1] == n_kv and t.shape[3] == dim,
                     f"out: two caches [{pages.shape[0]}, {n_kv}, rows, {dim}] in {self.dtype}")
        _ops().paged_load(k, v, ks, vs, pages, last_pos, k_out, v_out)
        return out
