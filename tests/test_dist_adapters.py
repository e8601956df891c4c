"""A prompt's adapter goes with its rows to every rank (gloo ranks on the CPU)."""
import os

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from nanochat_b200.dist import shard_rows, sharded_prefill
from nanochat_b200.engine import KVCache

from .test_dist_cpu import _free_port


def _worker(rank, world, port, slot, p, ret):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        from tests.cpu_backend import oracle_backend
        common = dict(num_heads=2, head_dim=16, num_layers=2, device="cpu", dtype=torch.float32)
        lo, hi = shard_rows(5, rank, world)
        prompt = None
        if rank == world - 1:  # the source is not always the first
            prompt = KVCache(batch_size=1, seq_len=9, **common)
            prompt.cache_seqlens.fill_(p)
            if slot is not None:
                prompt.adapter_slots = torch.tensor([slot], dtype=torch.int32)
        local = KVCache(batch_size=hi - lo, seq_len=20, **common)
        with oracle_backend():
            sharded_prefill(prompt, local, src=world - 1)
        slots = local.adapter_slots
        ret.put(slots is None if slot is None else slots is not None and slots.dtype == torch.int32 and slots.tolist() == [slot] * (hi - lo))
    finally:
        dist.destroy_process_group()


@pytest.mark.parametrize("slot,p", [(2, 9), (0, 0), (-1, 4), (None, 9)])
def test_every_rank_has_the_prompts_adapter(slot, p):
    ctx = mp.get_context("spawn")
    ret = ctx.Queue()
    port, world = _free_port(), 2
    procs = [ctx.Process(target=_worker, args=(r, world, port, slot, p, ret)) for r in range(world)]
    for pr in procs:
        pr.start()
    for pr in procs:
        pr.join(120)
        assert pr.exitcode == 0
    assert all(ret.get(timeout=10) for _ in range(world))
