"""One gloo rank of the tensor-parallel test of projections in 8 bits (started by tests/test_e4m3_model.py through torch.distributed.run): every schedule with
its shard of the weights, with stand-in operators, against the same arithmetic in 16 bits."""
import copy
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
from cpu_ops import CpuOps  # noqa: E402
from e4m3_ops import E4M3Ops, fake_weights, faked_ops  # noqa: E402
from oracle import ladder_oracle as lo  # noqa: E402
from test_paged_model import FAMILIES  # noqa: E402

from gpt_fast import e4m3  # noqa: E402


class Ops(E4M3Ops, CpuOps):
    pass


def main():
    rank, world = dist.get_rank(), dist.get_world_size()
    e4m3.CudaOps = E4M3Ops
    for family, (mod, cls) in FAMILIES.items():
        cfg = gu.tiny_config(family)
        full = lo.make_full_weights(cfg, gu.SEED, **gu.INITS["loud"])
        kw = gu.preset_kwargs(cfg)
        if family == "desync":
            kw["reduce_pattern"] = cfg.reduce_pattern
        mod.transformer_configs["tiny-e4m3"] = kw
        model = cls.from_name("tiny-e4m3").to(torch.bfloat16).eval()
        gu.load_shards(model, family, cfg, full, rank, world, torch.bfloat16)
        tokens = torch.randint(0, cfg.vocab_size, (2, 14), generator=torch.Generator().manual_seed(1))

        def run(ops):
            model.setup_caches(2, 32)
            model._engine.ops = ops
            out = [model(tokens[:, :11], torch.arange(11))]
            for s in range(11, 14):
                out.append(model(tokens[:, s:s + 1], torch.tensor([s])))
            return torch.cat(out, 1).float()

        eight = copy.deepcopy(model)
        fake_weights(model)
        want = run(faked_ops(cfg.vocab_size))  # the same arithmetic, but for roundings to bfloat16 that turn a code in twenty
        model = eight.quantize_projections()
        got = run(Ops)
        err = ((got - want).norm() / want.norm()).item()
        assert err < 0.25, f"{family} rank {rank}: {err}"
        if family != "desync":  # whose ranks may differ
            seen = [torch.empty_like(got) for _ in range(world)]
            dist.all_gather(seen, got.contiguous())
            assert all(torch.equal(s, got) for s in seen)
    dist.barrier()
    if rank == 0:
        print("E4M3-CPU-OK")


if __name__ == "__main__":
    with torch.no_grad():
        main()
