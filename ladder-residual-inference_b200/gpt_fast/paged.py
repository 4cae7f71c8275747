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

from ._C import ZERO_SKIPPED
from .ops import CudaOps

_E4M3 = torch.float8_e4m3fn


def _said(t):
    return f"{t.dtype} {tuple(t.shape)} with strides {t.stride()}"


def _check_rows(rows, input_pos, pages, pages_shape):
    dtype = input_pos.dtype
    if not ((dtype is torch.int32 or dtype is torch.int64) and input_pos.shape == (rows,) and input_pos.is_contiguous()):
        raise ValueError(f"positions: {rows} contiguous int32 or int64 numbers, not {_said(input_pos)}")
    if not (pages.dtype is torch.int32 and len(pages_shape) == 2 and pages_shape[1] >= 1 and
            (pages.is_contiguous() or pages.stride(1) == 1 <= pages.stride(0))):
        raise ValueError(f"pages: an int32 table [sequences, most pages] with contiguous rows, not {_said(pages)}")


def _check_like(out, dtype, shape):
    if not (out.dtype is dtype and out.shape == shape and out.is_contiguous()):
        raise ValueError(f"out: contiguous {dtype} {tuple(shape)}, not {_said(out)}")


class PagedKVCache(nn.Module):
    """k_pages, v_pages [n_pages, n_heads, page_size, head_dim] in `cache_dtype` (default: dtype), and k_scale, v_scale
    [n_pages, n_heads, page_size] where that is torch.float8_e4m3fn, None otherwise."""

    ops = CudaOps

    def __init__(self, n_pages: int, page_size: int, n_heads: int, head_dim: int, dtype: torch.dtype = torch.bfloat16,
                 cache_dtype: Optional[torch.dtype] = None, device=None):
        super().__init__()
        cache_dtype = dtype if cache_dtype is None else cache_dtype
        if dtype not in (torch.bfloat16, torch.float16):
            raise TypeError(f"a paged cache works with bfloat16 or float16 activations, not {dtype}")
        if cache_dtype not in (dtype, _E4M3):
            raise TypeError(f"pages hold the activations' type ({dtype}) or float8_e4m3fn, not {cache_dtype}")
        if n_pages < 1 or n_heads < 1:
            raise ValueError(f"{n_pages} pages of {n_heads} heads")
        if page_size % 8 or not 8 <= page_size <= 4096:
            raise ValueError(f"page_size={page_size}: a multiple of 8 up to 4096")
        if head_dim % 8 or not 8 <= head_dim <= 256:
            raise ValueError(f"head_dim={head_dim}: a multiple of 8 up to 256")
        self.dtype = dtype
        shape = (n_pages, n_heads, page_size, head_dim)
        self.register_buffer("k_pages", torch.zeros(shape, dtype=cache_dtype, device=device))
        self.register_buffer("v_pages", torch.zeros(shape, dtype=cache_dtype, device=device))
        self.register_buffer("k_scale", torch.zeros(shape[:3], device=device) if cache_dtype is _E4M3 else None)
        self.register_buffer("v_scale", torch.zeros(shape[:3], device=device) if cache_dtype is _E4M3 else None)

    def _tensors(self):
        """The four buffers, which a caller may have replaced; a module that was cast to another type after its caches were made holds codes
        without their meaning."""
        b = self._buffers
        k, v, ks, vs = b["k_pages"], b["v_pages"], b["k_scale"], b["v_scale"]
        dtype, shape = k.dtype, k.shape
        ok = dtype is v.dtype and len(shape) == 4 and shape == v.shape and k.is_contiguous() and v.is_contiguous()
        if ks is None:
            ok = ok and vs is None and dtype is self.dtype
        else:
            ok = (ok and vs is not None and dtype is _E4M3 and ks.dtype is vs.dtype is torch.float32 and ks.shape == vs.shape == shape[:3] and
                  ks.is_contiguous() and vs.is_contiguous())
        if not ok:
            raise ValueError(f"contiguous pages [n_pages, n_heads, page_size, head_dim] of {self.dtype} without scales, or of float8_e4m3fn with fp32 scales "
                             "[n_pages, n_heads, page_size]")
        return k, v, ks, vs, shape

    def store(self, qkv: Tensor, table: Optional[Tensor], input_pos: Tensor, pages: Tensor, n_head: int,
              sequence: Optional[Tensor] = None, halves: bool = False, out: Optional[Tensor] = None) -> Tensor:
        """qkv [tokens, (n_head + 2 n_heads) head_dim], rows [q | k | v heads] of the fused projection: rotates queries and keys by their
        positions, writes keys and values into the pages, returns the queries [tokens, n_head, head_dim].  Token i has position
        input_pos[i] in sequence sequence[i] (None: in sequence i).  table [positions, rot / 2, 2] (cos, sin) in the activations' type or
        fp32, None for no rotation: the first rot elements of a head turn, in adjacent pairs (utils.precompute_freqs_cis) or in halves.
        A token without a position (negative, behind the table) or without a page is left out: its query row is zeros, and in an `out` of the caller's
        stays as it was.  One call may name a (sequence, position) once."""
        k, v, ks, vs, cache_shape = self._tensors()
        _, n_kv, _, dim = cache_shape
        dtype, shape, pages_shape = self.dtype, qkv.shape, pages.shape
        if not (len(shape) == 2 and n_head >= 1 and shape[1] == (n_head + 2 * n_kv) * dim and qkv.dtype is dtype and
                (qkv.is_contiguous() or qkv.stride(1) == 1)):
            raise ValueError(f"qkv: rows of {n_head} + 2 * {n_kv} heads of {dim} in {dtype}, not {_said(qkv)}")
        tokens = shape[0]
        _check_rows(tokens, input_pos, pages, pages_shape)
        if not (tokens == pages_shape[0] if sequence is None else
                sequence.dtype is torch.int32 and sequence.shape == (tokens,) and sequence.is_contiguous()):
            raise ValueError(f"sequence: {tokens} contiguous int32 numbers, or None for one token of each of {pages_shape[0]} sequences")
        if table is not None:
            shape = table.shape
            if not (len(shape) == 3 and shape[2] == 2 and 2 <= 2 * shape[1] <= dim and table.is_contiguous() and
                    (table.dtype is dtype or table.dtype is torch.float32)):
                raise ValueError(f"table: [positions, rot / 2, 2] in {dtype} or float32, rot up to {dim}, not {_said(table)}")
        args = n_head, bool(halves), tokens, pages_shape, cache_shape
        if out is None:
            out = qkv.new_empty((tokens, n_head, dim))
            self.ops.rope_paged_store(qkv, table, input_pos, sequence, pages, out, k, v, ks, vs, *args, ZERO_SKIPPED)
        else:
            _check_like(out, dtype, (tokens, n_head, dim))
            self.ops.rope_paged_store(qkv, table, input_pos, sequence, pages, out, k, v, ks, vs, *args)
        return out

    def attend_workspace(self, n_head: int) -> Tensor:
        """The workspace of `attend`: shared by calls that do not overlap on the device, and kept by the caller as long as graphs captured with it."""
        k = self.k_pages
        return torch.zeros(self.ops.paged_attn_workspace_bytes(n_head, k.shape[1], k.shape[3]), dtype=torch.uint8, device=k.device)

    def attend(self, q: Tensor, input_pos: Tensor, pages: Tensor, window: int = 0, scale: Optional[float] = None,
               out: Optional[Tensor] = None, workspace: Optional[Tensor] = None) -> Tensor:
        """Attention of one new token of each sequence, whose row is in the cache: q [sequences, n_head, head_dim] over positions
        0 .. input_pos[b] (the last `window` of them if it is not 0); zeros where that is none.  scale: 1 / sqrt(head_dim) by default.
        workspace: from attend_workspace(n_head); allocated for the call if None."""
        k, v, ks, vs, cache_shape = self._tensors()
        _, n_kv, _, dim = cache_shape
        shape, pages_shape = q.shape, pages.shape
        if not (len(shape) == 3 and q.dtype is self.dtype and q.is_contiguous() and shape[2] == dim and shape[1] >= 1 and shape[1] % n_kv == 0):
            raise ValueError(f"q: contiguous [sequences, a multiple of {n_kv}, {dim}] in {self.dtype}, not {_said(q)}")
        n_seq, n_head, _ = shape
        _check_rows(n_seq, input_pos, pages, pages_shape)
        if pages_shape[0] != n_seq:
            raise ValueError(f"pages of {pages_shape[0]} sequences for {n_seq}")
        if not 0 <= window < 1 << 62:
            raise ValueError(f"window={window}")
        if workspace is None:
            workspace = self.attend_workspace(n_head)
        elif not (workspace.dtype is torch.uint8 and workspace.is_contiguous()):
            raise ValueError(f"workspace: bytes from attend_workspace, not {_said(workspace)}")
        if out is None:
            out = torch.empty_like(q)
        else:
            _check_like(out, q.dtype, shape)
        self.ops.paged_attention(q, k, v, ks, vs, pages, input_pos, window, dim ** -0.5 if scale is None else scale, out, workspace, n_head, pages_shape,
                                 cache_shape)
        return out

    def load(self, last_pos: Tensor, pages: Tensor, rows: Optional[int] = None, out: Optional[Tuple[Tensor, Tensor]] = None):
        """Positions 0 .. last_pos[b] of every sequence as dense caches (k, v) [sequences, n_heads, rows, head_dim] in the activations'
        type, as KVCache holds them: what prompt attention works on.  `out` is written in place: rows behind the last position up to
        a multiple of 64 become zeros, later ones stay as they were.  Without it caches of `rows` positions (default: all that the
        table's pages hold) are made, zero behind the last position."""
        k, v, ks, vs, cache_shape = self._tensors()
        _, n_kv, page, dim = cache_shape
        pages_shape = pages.shape
        n_seq = pages_shape[0] if len(pages_shape) else 0
        _check_rows(n_seq, last_pos, pages, pages_shape)
        if out is None:
            shape = (n_seq, n_kv, pages_shape[1] * page if rows is None else rows, dim)
            out = torch.zeros(shape, dtype=self.dtype, device=k.device), torch.zeros(shape, dtype=self.dtype, device=k.device)
        k_out, v_out = out
        rows = k_out.shape[2] if k_out.dim() == 4 else -1
        shape = (n_seq, n_kv, rows, dim)
        _check_like(k_out, self.dtype, shape)
        _check_like(v_out, self.dtype, shape)
        self.ops.paged_load(k, v, ks, vs, pages, last_pos, k_out, v_out, rows, pages_shape, cache_shape)
        return out
