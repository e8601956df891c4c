"""Counts of new tokens that cannot be: flagged, and the cache moves by what was written."""
import pytest
import torch

from nanochat_b200 import ops
from nanochat_b200.gpt import kv_attention, precompute_rotary_embeddings


class Pages:
    paged, n_layers = True, 1

    def __init__(self, lens):
        self.cache_seqlens = torch.tensor(lens, dtype=torch.int32)
        self.block_table = torch.zeros(len(lens), 1, dtype=torch.int32)

    def get_layer_cache(self, layer):
        return None, None

    def advance(self, n):
        self.cache_seqlens += n


def test_lengths_move_by_what_was_written(monkeypatch):
    monkeypatch.setattr(ops, "append_rope_norm_paged", lambda q, *a, **k: q)
    monkeypatch.setattr(ops, "prefill_attention_paged", lambda q, *a: q)
    monkeypatch.setattr(ops, "append_and_attend", lambda *a: None)
    cache, x = Pages([10, 20, 30, 40]), torch.zeros(4, 3, 1, 128)
    kv_attention(x, x, x, (None, None), (-1, 0), cache, 0, new_tokens=torch.tensor([4, -1, 3, 0], dtype=torch.int32))
    assert cache.cache_seqlens.tolist() == [13, 20, 33, 40] and cache.cache_seqlens.dtype == torch.int32
    kv_attention(x, x, x, (None, None), (-1, 0), cache, 0)
    assert cache.cache_seqlens.tolist() == [16, 23, 36, 43]


@pytest.mark.gpu
def test_the_next_step_behind_counts_that_cannot_be():
    from .test_chunk_pages_gpu import caches
    B, T, Hq, Hkv, page = 3, 5, 4, 2, 48
    tables = precompute_rotary_embeddings(240, 128, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(2)
    first, second = ([torch.randn(B, n, h, 128, generator=gen, device="cuda").bfloat16() for h in (Hq, Hkv, Hkv)] for n in (T, 2))
    got = []
    for counts in ([T + 1, -1, 2], [T, 0, 2]):
        _, cache = caches(B, Hkv, 1, 240, page)
        cache.reserve(48)
        y = kv_attention(*first, tables, (-1, 0), cache, 0, new_tokens=torch.tensor(counts, dtype=torch.int32, device="cuda"))
        assert ops.read_status("cuda") == (5 if counts[1] < 0 else 0)
        got.append((y, cache.cache_seqlens.tolist(), kv_attention(*second, tables, (-1, 0), cache, 0)))
    assert got[0][1] == [T, 0, 2] and got[0][1] == got[1][1]
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][2], got[1][2])
