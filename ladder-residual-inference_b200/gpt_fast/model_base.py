"""Pieces shared by the four family modules: ModelArgs, the model shell and the block shell.

The reference repeats these in every family file (gpt_fast/gpt_ladder_TP.py:20-62, 210-288 and
its three siblings); here the family files keep only what differs between schedules.
"""
from dataclasses import dataclass
from typing import Optional

import torch
import torch.distributed as dist
import torch.nn as nn
from torch import Tensor

from .e4m3 import E4M3Linear
from .engine import Engine
from .paged import PagedKVCache
from .utils import KVCache, RMSNorm, precompute_freqs_cis


def find_multiple(n: int, k: int) -> int:
    return n if n % k == 0 else n + k - (n % k)


@dataclass
class ModelArgsBase:
    block_size: int = 2048
    vocab_size: int = 32000
    n_layer: int = 32
    n_head: int = 32
    dim: int = 4096
    intermediate_size: int = None
    n_local_heads: int = -1
    head_dim: int = 64
    rope_base: float = 10000
    norm_eps: float = 1e-5
    rope_scaling: Optional[dict] = None
    semi_compiled_model: bool = False

    def __post_init__(self):
        world = dist.get_world_size()
        if self.n_local_heads == -1:
            self.n_local_heads = self.n_head
        if self.intermediate_size is None:
            # the usual Llama rule: 2/3 of 4*dim, rounded up to a multiple of 256
            self.intermediate_size = find_multiple(int(2 * (4 * self.dim) / 3), 256)
        self.head_dim = self.dim // self.n_head
        assert self.dim % world == 0
        assert self.intermediate_size % world == 0


def args_from_name(cls, table, name):
    if name not in table:
        raise KeyError(f"unknown preset {name!r}; known presets: {sorted(table)}")
    return cls(**table[name])


class TPModelBase(nn.Module):
    """tok_embeddings, layers, norm, output (replicated LM head), freqs_cis, causal_mask,
    max_batch_size, max_seq_length: the attributes the benchmark driver and the reference's own
    code use.  forward(idx [B, S], input_pos [S]) -> logits [B, S, vocab]."""

    family = ""
    engine_class = Engine
    dtypes = (torch.bfloat16, torch.float16)  # storage types the family's kernels run

    def __init__(self, config, blocks) -> None:
        super().__init__()
        self.config = config
        self.tok_embeddings = nn.Embedding(config.vocab_size, config.dim)
        self.layers = nn.ModuleList(blocks)
        self.norm = RMSNorm(config.dim, eps=config.norm_eps)
        self.output = nn.Linear(config.dim, config.vocab_size, bias=False)
        self.freqs_cis: Optional[Tensor] = None
        self.mask_cache: Optional[Tensor] = None
        self.max_batch_size = -1
        self.max_seq_length = -1
        self._engine = None

    def setup_caches(self, max_batch_size, max_seq_length):
        if self.max_seq_length >= max_seq_length and self.max_batch_size >= max_batch_size and not self._engine.paged:
            return
        max_seq_length = find_multiple(max_seq_length, 8)
        self.max_seq_length = max_seq_length
        self.max_batch_size = max_batch_size
        dtype = self.output.weight.dtype
        device = self.output.weight.device
        self._setup_layer_caches(max_batch_size, max_seq_length, dtype, device)
        self._engine = self.engine_class(self, self.family)
        self._engine.setup(max_batch_size, max_seq_length, device, dtype)

    def quantize_projections(self):
        """The layers' projections from here on in 8 bits: weights as e4m3 codes with a scale for each output, activations brought to e4m3 with a
        scale for each row by the norms in front of them (gpt_fast.e4m3).  Half the bytes of the layers for a decode step, twice the rate of
        the tensor cores for a prompt; embedding, norms, caches, attention and output projection stay as they are.  To be called with the
        weights in place, on their GPU, before caches are set up.  No counterpart in the reference."""
        if self.engine_class is not Engine:
            raise TypeError(f"the layers of {type(self).__name__} keep their projections in 16 bits")
        if self._engine is not None:
            raise RuntimeError("projections go to 8 bits before caches are set up")
        found = [(part, name, module) for block in self.layers for part in (block.attention, getattr(block, "feed_forward", None)) if part is not None
                 for name, module in part.named_children() if isinstance(module, nn.Linear)]
        for _, name, module in found:  # (all of them before the first is replaced)
            try:
                E4M3Linear.check(module)
            except ValueError as e:
                raise ValueError(f"{name}: {e}") from None
        if len({module.weight.device for _, _, module in found}) > 1:
            raise ValueError("the layers' projections are on several devices")
        while found:
            part, name, module = found.pop(0)
            setattr(part, name, E4M3Linear(module.weight))
            del module  # (a weight of 16 bits goes as soon as it has been read: a model may fill more than half of the memory)
        return self

    def _setup_layer_caches(self, max_batch_size, max_seq_length, dtype, device):
        cfg = self.config
        head_dim = cfg.dim // cfg.n_head
        for b in self.layers:
            b.attention.kv_cache = KVCache(max_batch_size, max_seq_length, cfg.n_local_heads // dist.get_world_size(),
                                           head_dim, dtype).to(device)
        self._setup_table(dtype, device)
        # kept because callers of the reference may read it; the kernels derive causality from input_pos
        self.causal_mask = torch.tril(torch.ones(max_seq_length, max_seq_length, dtype=torch.bool, device=device))

    def setup_paged_caches(self, max_sequences, n_pages, page_size=32, max_length=None, max_prompt=None, cache_dtype=None):
        """Caches in pages, for sequences of unequal lengths that come and go: the calls below then take `pages`, an int32 table [sequences, most
        pages] on the device that names each sequence's pages in order (-1: none), and a position for every token: a step of up to max_sequences
        new tokens (idx [B, 1], input_pos [B]; -1 for an idle row), or a prompt of one sequence, whole or in portions of up to max_prompt tokens
        (512 by default, or max_length; idx [1, S], input_pos [S], -1 for padding, pages [1, most pages]). max_length: the most positions of a
        sequence, the model's block_size by default (a prompt whose row of the table names more makes a larger copy of its pages to work on).
        cache_dtype: the model's type, or torch.float8_e4m3fn. A new token sees the positions up to its own that have a page, in a prompt as in a
        step. A token whose position has no page, or lies behind the table's pages or the model's block_size, is not stored; its logits mean
        nothing, but come from this call and the sequence's pages alone. No counterpart in the reference, whose sequences share their positions
        (gpt_fast/gpt_ladder_TP.py:252-284)."""
        if self.engine_class is not Engine:
            raise TypeError(f"the layers of {type(self).__name__} keep caches of their own kinds, not pages")
        cfg = self.config
        max_length = cfg.block_size if max_length is None else max_length
        assert 1 <= max_length <= cfg.block_size, f"max_length={max_length}: 1 to the model's block_size, {cfg.block_size}"
        max_prompt = min(512, max_length) if max_prompt is None else max_prompt
        assert 1 <= max_prompt <= max_length, f"max_prompt={max_prompt}: 1 to max_length, {max_length}"
        dtype, device, head_dim = self.output.weight.dtype, self.output.weight.device, cfg.dim // cfg.n_head
        for b in self.layers:
            b.attention.kv_cache = PagedKVCache(n_pages, page_size, cfg.n_local_heads // dist.get_world_size(), head_dim, dtype, cache_dtype, device)
        self.max_batch_size, self.max_seq_length = max_sequences, max_length
        self._setup_table(dtype, device)
        self._engine = self.engine_class(self, self.family)
        self._engine.setup_paged(max_sequences, max_prompt, max_length, device, dtype)

    def _setup_table(self, dtype, device):
        cfg = self.config
        self.freqs_cis = precompute_freqs_cis(cfg.block_size, cfg.dim // cfg.n_head, cfg.rope_base, dtype,
                                              cfg.rope_scaling).to(device).contiguous()

    def recurrent_state(self):
        """Tensors a step reads and overwrites, so that repeating a step needs them restored (none for attention
        caches: rewriting a position with the same values changes nothing)."""
        return []

    def forward(self, idx: Tensor, input_pos: Optional[Tensor] = None, pages: Optional[Tensor] = None) -> Tensor:
        assert self._engine is not None, "Caches must be initialized first"
        return self._engine.forward(idx, input_pos, pages)

    def prefill_last(self, idx: Tensor, input_pos: Tensor, pages: Optional[Tensor] = None) -> Tensor:
        """forward(idx, input_pos)[:, -1:] without computing the other positions' logits (no
        counterpart in the reference, whose forward always projects every position)."""
        assert self._engine is not None, "Caches must be initialized first"
        return self._engine.forward_last(idx, input_pos, pages)

    def decode_greedy(self, idx: Tensor, input_pos: Tensor, pages: Optional[Tensor] = None) -> Tensor:
        """Arg-max next token of every sequence, int32 [B, 1]; equal to
        `forward(idx, input_pos)[:, -1].argmax(-1)` but with the output projection split by
        vocabulary over the tensor-parallel ranks (no counterpart in the reference, which
        samples from the replicated logits, benchmark.py:74-92)."""
        assert self._engine is not None, "Caches must be initialized first"
        return self._engine.forward_greedy(idx, input_pos, pages)

    def decode_sample(self, idx: Tensor, input_pos: Tensor, temperature: float = 1.0, top_k: Optional[int] = None,
                      generator=None, pages: Optional[Tensor] = None) -> Tensor:
        """One sampled next token per sequence, int32 [B, 1], by the reference's rule
        (`sample(model(idx, input_pos), temperature, top_k)[0]`, benchmark.py:56-92), computed on the
        vocabulary-split output projection; see Engine.forward_sample."""
        assert self._engine is not None, "Caches must be initialized first"
        return self._engine.forward_sample(idx, input_pos, temperature, top_k, generator, pages)


class BlockBase(nn.Module):
    def extra_repr(self) -> str:
        return f"semi_compiled = {self.semi_compiled_model}"
