"""What a captured decode step reads of its cache when that was replaced between two steps (host logic with a stand-in for the graph, then the GPU)."""
import contextlib
from types import SimpleNamespace

import pytest
import torch

from nanochat_b200.engine import GraphedDecodeStep, KVCache


class Model:
    """Notes the tensors that a pass reads: what a graph would go on reading."""

    def __init__(self):
        self.adapters = SimpleNamespace(slots=4)

    def forward(self, ids, kv_cache):
        self.slots, self.prev = kv_cache.adapter_slots, kv_cache.prev_embedding
        kv_cache.prev_embedding = torch.ones_like(self.prev)
        return torch.zeros(ids.size(0), 1, 3)


@pytest.fixture
def no_cuda(monkeypatch):
    stream = SimpleNamespace(wait_stream=lambda other: None, synchronize=lambda: None)
    for name, value in dict(Stream=lambda dev=None: stream, current_stream=lambda dev=None: stream, stream=lambda s: contextlib.nullcontext(),
                            CUDAGraph=lambda: SimpleNamespace(replay=lambda: None), graph=lambda g, stream=None: contextlib.nullcontext()).items():
        monkeypatch.setattr(torch.cuda, name, value)


def captured(slots):
    cache = KVCache(batch_size=2, num_heads=1, seq_len=8, head_dim=128, num_layers=1, device="cpu", dtype=torch.float32)
    cache.prev_embedding = torch.full((2, 1, 4), 5.0)
    cache.adapter_slots = slots
    model, ids = Model(), torch.zeros(2, 1, dtype=torch.long)
    return cache, model, ids, GraphedDecodeStep(model, cache, ids)


def ints(*values):
    return torch.tensor(values, dtype=torch.int32)


def test_slots_that_were_replaced_or_written(no_cuda):
    mine = ints(1, 2)
    cache, model, ids, step = captured(mine)
    assert cache.adapter_slots is mine
    step.step(ids)
    assert model.slots.tolist() == [1, 2]
    cache.adapter_slots = ints(3, -1)
    step.step(ids)
    assert model.slots.tolist() == [3, -1] and mine.tolist() == [1, 2]
    cache.adapter_slots[0] = 0
    step.step(ids)
    assert model.slots.tolist() == [0, -1]
    cache.adapter_slots = None  # as reset() leaves it
    step.step(ids)
    assert model.slots.tolist() == [-1, -1]


def test_what_a_captured_step_cannot_follow(no_cuda):
    cache, model, ids, step = captured(ints(1, 2))
    for bad in (ints(1), ints(1, 2).long(), ints(1, 2).view(2, 1)):
        cache.adapter_slots = bad
        with pytest.raises(RuntimeError, match="adapter_slots"):
            step.step(ids)
    cache.adapter_slots, model.adapters = ints(1, 2), SimpleNamespace(slots=4)
    with pytest.raises(RuntimeError, match="bank"):
        step.step(ids)
    cache, model, ids, step = captured(None)
    step.step(ids)
    cache.adapter_slots = ints(0, 0)
    with pytest.raises(RuntimeError, match="without"):
        step.step(ids)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["dense", "paged"])
def test_a_captured_step_with_other_adapters(kind):
    from .test_adapters_model_gpu import cache_of, make
    m, _ = make()
    ids = torch.randint(0, 512, (3, 20), generator=torch.Generator().manual_seed(2)).cuda()
    caches = [cache_of(kind, 3, [1, -1, 0]) for _ in range(2)]
    for cache in caches:
        m.forward(ids[:, :10], kv_cache=cache)
    step = GraphedDecodeStep(m, caches[0], ids[:, 10:11])
    for at, slots in ((10, [1, -1, 0]), (11, [0, 1, -1]), (12, None), (13, [-1, -1, 1])):
        for cache in caches:
            cache.adapter_slots = None if slots is None else torch.tensor(slots, dtype=torch.int32, device="cuda")
            torch.full((1024,), 1, dtype=torch.int32, device="cuda")  # what was freed is somebody else's
        got = step.step(ids[:, at:at + 1])
        assert torch.equal(got, m.forward(ids[:, at:at + 1], kv_cache=caches[1])[:, -1])


def test_a_smear_state_that_was_replaced(no_cuda):
    """By a chunk into the cache between two steps, by drafts that were taken back, by reset()."""
    cache, model, ids, step = captured(None)
    step.step(ids)
    assert model.prev.eq(5).all()  # (the stand-in's replay writes nothing)
    cache.prev_embedding = torch.full((2, 1, 4), 7.0)
    step.step(ids)
    assert model.prev.eq(7).all() and cache.prev_embedding is model.prev
    cache.prev_embedding = None
    step.step(ids)
    assert model.prev.eq(0).all() and cache.prev_embedding is model.prev


@pytest.mark.gpu
def test_chunks_into_pages_between_captured_steps():
    from nanochat_b200 import ops
    from nanochat_b200.engine import PagedKVCache
    from .test_chunks_behind_tokens import cache_of, make
    m = make("cuda", torch.bfloat16, 256, 2, 1)
    ids = torch.randint(0, 128, (2, 40), generator=torch.Generator().manual_seed(6)).cuda()
    caches = [cache_of(PagedKVCache, m, 2, page_tokens=48) for _ in range(2)]
    for cache in caches:
        cache.reserve(48)
        m.forward(ids[:, :8], kv_cache=cache)
    step = GraphedDecodeStep(m, caches[0], ids[:, 8:9])
    for lo, hi in ((8, 9), (9, 10), (10, 15), (15, 16), (16, 18), (18, 19), (19, 20)):
        want = m.forward(ids[:, lo:hi], kv_cache=caches[1])[:, -1]
        got = step.step(ids[:, lo:hi]) if hi == lo + 1 else m.forward(ids[:, lo:hi], kv_cache=caches[0])[:, -1]
        assert torch.equal(got, want), (lo, hi)
    assert ops.read_status("cuda") == 0


def test_a_pass_that_is_refused_leaves_the_cache_as_it_was():
    from nanochat_b200.adapters import AdapterBank
    from nanochat_b200.gpt import GPT, GPTConfig
    m = GPT(GPTConfig(sequence_len=64, vocab_size=64, n_layer=1, n_head=2, n_kv_head=1, n_embd=256))
    m.init_weights()
    cache = KVCache(batch_size=2, num_heads=1, seq_len=8, head_dim=128, num_layers=1, device="cpu", dtype=torch.float32)
    prev = cache.prev_embedding = torch.zeros(2, 1, 256)
    cache.adapter_slots = ints(0, 0)
    ids = torch.zeros(2, 1, dtype=torch.long)
    with pytest.raises(ValueError, match="bank"):
        m.forward(ids, kv_cache=cache)
    m.adapters = AdapterBank(m, 1, 8)
    for bad in (ints(0), ints(0, 0).long(), ints(0, 0).to("meta"), ints(0, 0, 0)[::2]):
        cache.adapter_slots = bad
        with pytest.raises(ValueError, match="adapter_slots"):
            m.forward(ids, kv_cache=cache)
    assert cache.prev_embedding is prev and cache.cache_seqlens.tolist() == [0, 0]
