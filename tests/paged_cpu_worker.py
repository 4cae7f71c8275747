"""One gloo rank of the paged tensor-parallel test (started by tests/test_paged_ranks.py through torch.distributed.run): every schedule with its shard of the
weights, on pages and on dense caches, with stand-in operators; prompts of unequal lengths, then steps of all sequences together."""
import os
import sys

import torch
import torch.distributed as dist

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
for p in (HERE, ROOT, os.path.join(ROOT, "ladder-residual-inference_b200")):
    sys.path.insert(0, p)

dist.init_process_group("gloo")

import golden_util as gu  # noqa: E402
from oracle import ladder_oracle as lo  # noqa: E402
from test_paged_left_out import Ops  # noqa: E402
from test_paged_model import FAMILIES  # noqa: E402

from gpt_fast.paged import PagedKVCache  # noqa: E402

PROMPTS, STEPS, PAGE = [19, 1, 8], 3, 8


def main():
    rank, world = dist.get_rank(), dist.get_world_size()
    PagedKVCache.ops = Ops
    for family, (mod, cls) in FAMILIES.items():
        cfg = gu.tiny_config(family)
        full = lo.make_full_weights(cfg, gu.SEED, **gu.INITS["loud"])
        kw = gu.preset_kwargs(cfg)
        if family == "desync":
            kw["reduce_pattern"] = cfg.reduce_pattern
        mod.transformer_configs["tiny-paged"] = kw
        model = cls.from_name("tiny-paged").to(torch.bfloat16).eval()
        gu.load_shards(model, family, cfg, full, rank, world, torch.bfloat16)
        tokens = torch.randint(0, cfg.vocab_size, (len(PROMPTS), max(PROMPTS) + STEPS), generator=torch.Generator().manual_seed(1))

        want = [[] for _ in PROMPTS]
        for b, n in enumerate(PROMPTS):
            model.max_seq_length = -1  # fresh caches
            model.setup_caches(1, 32)
            model._engine.ops = Ops
            want[b].append(model(tokens[b:b + 1, :n], torch.arange(n))[0])
            for s in range(STEPS):
                want[b].append(model(tokens[b:b + 1, n + s:n + s + 1], torch.tensor([n + s]))[0])

        model.setup_paged_caches(len(PROMPTS), 12, PAGE, max_length=32, max_prompt=24)
        model._engine.ops = Ops
        assert tuple(model.layers[0].attention.kv_cache.k_pages.shape) == (12, cfg.n_local_heads // world, PAGE, cfg.head_dim)
        table = torch.full((3, 4), -1, dtype=torch.int32)
        table[0, :3], table[1, :1], table[2, :2] = torch.tensor([7, 0, 11]), torch.tensor([3]), torch.tensor([5, 2])
        got = [[] for _ in PROMPTS]
        for b, n in enumerate(PROMPTS):
            got[b].append(model(tokens[b:b + 1, :n], torch.arange(n), table[b:b + 1])[0])
        for s in range(STEPS):
            idx = torch.stack([tokens[b, n + s] for b, n in enumerate(PROMPTS)])[:, None]
            pos = torch.tensor([n + s for n in PROMPTS], dtype=torch.int32)
            logits = model(idx, pos, table)
            chosen = model.decode_greedy(idx, pos, table)
            for b in range(len(PROMPTS)):
                got[b].append(logits[b])
            if family != "desync":  # whose ranks may differ
                assert torch.equal(chosen[:, 0].long(), logits[:, -1].float().argmax(-1))
        for b in range(len(PROMPTS)):
            # both in bf16 with the same roundings: sums differ in the last place of 32 bits at most, which may turn a rounding now and then
            g, w = torch.cat(got[b]).float(), torch.cat(want[b]).float()
            err = ((g - w).norm() / w.norm()).item()
            assert err < 1e-2, f"{family} rank {rank} sequence {b}: {err}"
    dist.barrier()
    if rank == 0:
        print("PAGED-CPU-OK")


if __name__ == "__main__":
    with torch.no_grad():
        main()
