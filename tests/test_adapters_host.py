"""A bank of adapters and where it is refused (no GPU)."""
import pytest
import torch

from nanochat_b200.adapters import AdapterBank
from nanochat_b200.engine import Engine, KVCache
from nanochat_b200.gpt import GPT, GPTConfig


def model(n_embd=256, heads=2):
    return GPT(GPTConfig(sequence_len=64, vocab_size=64, n_layer=2, n_head=heads, n_kv_head=1, n_embd=n_embd))


def pair(bank, name, rank):
    layer, part = int(name.split(".")[2]), name.split(".", 3)[3]
    down, up = bank.layers[layer][part]
    return {name + ".down": torch.randn(rank, down.size(2)), name + ".up": torch.randn(up.size(1), rank)}


def test_load_and_clear():
    m = model()
    bank = AdapterBank(m, slots=3, rank=12)
    assert m.adapters is bank and bank.layers[0]["attn.c_k"][0].shape == (3, 16, 256) and bank.layers[1]["mlp.c_fc"][1].shape == (3, 1024, 16)
    name = "transformer.h.1.mlp.c_proj"
    tensors = {**pair(bank, name, 5), **pair(bank, "transformer.h.0.attn.c_q", 12)}
    bank.load(2, tensors, scale=0.25)
    down, up = bank.layers[1]["mlp.c_proj"]
    assert torch.equal(down[2, :5], tensors[name + ".down"].bfloat16()) and not down[2, 5:].any() and not down[:2].any()
    assert torch.equal(up[2, :, :5], tensors[name + ".up"].bfloat16()) and not up[2, :, 5:].any()
    assert bank.scales.tolist() == [0, 0, 0.25]
    bank.load(2, pair(bank, name, 1), scale=2)  # the one before is gone
    assert not bank.layers[0]["attn.c_q"][0].any() and not down[2, 1:].any()
    bank.clear(2)
    assert not down.any() and not up.any() and not bank.scales.any()
    some = AdapterBank(m, 1, 8, projections=("attn.c_v",))
    assert set(some.layers[0]) == {"attn.c_v"} and some.at(0, None)("mlp.c_fc", 1, 2) == 1


def test_refusals():
    m = model()
    for slots, rank in ((0, 8), (2, 0), (2, 129)):
        with pytest.raises(ValueError):
            AdapterBank(m, slots, rank)
    for projections in ((), ("lm_head",), ("attn.c_q", "attn.ve_gate")):
        with pytest.raises(ValueError):
            AdapterBank(m, 2, 8, projections)
    bank = AdapterBank(m, 2, 8, projections=("attn.c_q",))
    name = "transformer.h.0.attn.c_q"
    good = pair(bank, name, 4)
    bank.load(0, good, scale=3)
    bad = [{name + ".down": good[name + ".down"]}, {**good, name + ".up": good[name + ".up"][:, :3]}, pair(bank, name, 9), {**good, name + ".bias": good[name + ".up"]},
           {"transformer.h.0.mlp.c_fc.down": good[name + ".down"]}, {"transformer.h.2.attn.c_q.down": good[name + ".down"]},
           {**good, name + ".down": good[name + ".down"][:, :8]}]
    for tensors in bad:
        with pytest.raises(ValueError):
            bank.load(0, tensors)
    assert bank.scales[0] == 3 and bank.layers[0]["attn.c_q"][0][0, :4].any()
    for slot in (-1, 2):
        with pytest.raises(ValueError):
            bank.load(slot, good)
        with pytest.raises(ValueError):
            bank.clear(slot)


def test_slots_follow_a_prompt_and_leave_with_it():
    common = dict(num_heads=1, seq_len=8, head_dim=128, num_layers=1, device="cpu", dtype=torch.float32)
    cache = KVCache(batch_size=1, **common)
    assert cache.adapter_slots is None
    cache.adapter_slots = torch.tensor([2], dtype=torch.int32)
    from nanochat_b200.engine import _broadcast_adapter
    rows = KVCache(batch_size=3, **common)
    _broadcast_adapter(rows, cache)
    assert rows.adapter_slots.tolist() == [2, 2, 2]
    rows.reset()
    assert rows.adapter_slots is None


def test_a_model_without_the_bank_refuses():
    m = model()
    cache = KVCache(batch_size=1, num_heads=1, seq_len=8, head_dim=128, num_layers=2, device="cpu", dtype=torch.float32)
    cache.adapter_slots = torch.zeros(1, dtype=torch.int32)
    m.init_weights()
    with pytest.raises(ValueError, match="bank"):
        m.forward(torch.zeros(1, 3, dtype=torch.long), kv_cache=cache)

    m.adapters = AdapterBank(m, 1, 8)
    cache.adapter_slots = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="each of 1 rows"):
        m.forward(torch.zeros(1, 3, dtype=torch.long), kv_cache=cache)
    m.adapters = None

    class Tokenizer:
        def encode_special(self, s):
            return 1

        def get_bos_token_id(self):
            return 0
    with pytest.raises(ValueError, match="no adapter"):
        next(Engine(m, Tokenizer()).generate([1, 2], adapter=0))


def test_the_operator_needs_the_gpu():
    from nanochat_b200 import ops
    t = torch.zeros(1, 1, 8, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.add_adapters(t, t, torch.zeros(1, 8, 8, dtype=torch.bfloat16), torch.zeros(1, 8, 8, dtype=torch.bfloat16),
                         torch.zeros(1, dtype=torch.int32), torch.ones(1))
    pool = torch.zeros(1, 48, 1, 128, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.prefill_attention_paged(torch.zeros(1, 2, 1, 128, dtype=torch.bfloat16), pool, pool, torch.zeros(1, 1, dtype=torch.int32),
                                    torch.zeros(1, dtype=torch.int32))
